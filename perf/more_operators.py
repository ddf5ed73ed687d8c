"""What the 8-bit paged cache and the sparse attention over it are measured on: cases over their range of use, their plain forms
and 64-bit values.

Four operators, parts of one path (a session's rows are written into a cache in 8 bits, read back or attended there; in long
sessions the queries attend only to blocks that a cheap score selects):

``pack``    rows quantised as they are written into pages: e4m3 codes, one e8m0 scale for each token and head; with or without
            the rotation of q and k on the way
``read``    rows of sessions out of such pages, dense and in 16 bits
``packed``  attention of new tokens over such pages, single tokens and chunks, with its log-sum-exp
``sparse``  means of the keys of the blocks that new tokens touched, the choice of blocks for every query block and KV head, and
            attention over the chosen ones, in 16-bit or 8-bit pages
"""

import functools
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
THETA = 10000.0
GRID = (30, 52)  # latent rows and columns of a frame: 1,560 tokens
LOW, HIGH = {"bf16": -124, "fp16": -15}, {"bf16": 119, "fp16": 7}  # exponents of scales: code * scale is a number of the type


# -- cases ------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one decoding step of 61 sessions: a token each into pages of 16
        dict(name="pack_step", op="pack", seqs=61, new=1, history=4096, heads=32, kv_heads=8, dim=128, page=16, layout="halves",
             dtype="fp16", ragged=False),
        # a chunk of three latent frames for each of three sessions, one frame to a page
        dict(name="pack_chunk", op="pack", seqs=3, new=4680, history=9360, heads=12, kv_heads=12, dim=128, page=1560,
             layout="interleaved", dtype="bf16", ragged=False),
        # rows that a norm kernel has rotated already, sessions of different lengths
        dict(name="pack_rows", op="pack", seqs=7, new=777, history=1000, heads=0, kv_heads=4, dim=64, page=24, layout="none",
             dtype="bf16", ragged=True),
        # five chunks of a session back into a contiguous cache
        dict(name="read_session", op="read", seqs=1, kv=23400, kv_heads=12, dim=128, page=1560, dtype="bf16", ragged=False),
        # short histories of many sessions, for an archive
        dict(name="read_many", op="read", seqs=40, kv=1500, kv_heads=8, dim=64, page=16, dtype="fp16", ragged=True),
        # one token of one session: latency
        dict(name="packed_token", op="packed", seqs=1, new=1, kv=2048, heads=32, kv_heads=8, dim=128, page=16, causal=True,
             dtype="bf16", ragged=False),
        # a decoding step of 48 sessions of very different lengths
        dict(name="packed_step", op="packed", seqs=48, new=1, kv=16384, heads=32, kv_heads=8, dim=128, page=64, causal=True,
             dtype="bf16", ragged=True),
        # a chunk of three latent frames that sees itself and four chunks before it
        dict(name="packed_chunk", op="packed", seqs=1, new=4680, kv=23400, heads=12, kv_heads=12, dim=128, page=1560, causal=False,
             dtype="bf16", ragged=False),
        # one token of one long session
        dict(name="sparse_token", op="sparse", seqs=1, new=1, kv=65536, heads=32, kv_heads=8, dim=128, page=64, block=64, keep=32,
             query_block=1, sinks=64, recent=128, causal=True, packed=False, dtype="bf16", ragged=False),
        # a decoding step of 40 sessions of very different lengths, in 8 bits
        dict(name="sparse_step", op="sparse", seqs=40, new=1, kv=32768, heads=32, kv_heads=8, dim=128, page=128, block=64, keep=24,
             query_block=1, sinks=4, recent=256, causal=True, packed=True, dtype="bf16", ragged=True),
        # pieces of prompts of four sessions, each a different length, after histories of different lengths
        dict(name="sparse_prompts", op="sparse", seqs=4, new=1021, kv=16000, heads=32, kv_heads=8, dim=128, page=64, block=32,
             keep=40, query_block=32, sinks=32, recent=64, causal=True, packed=False, dtype="fp16", ragged=True),
        # a chunk of three latent frames late in a long session: itself, a sink frame and 48 blocks for every 128 of its tokens
        dict(name="sparse_chunk", op="sparse", seqs=1, new=4680, kv=46800, heads=10, kv_heads=10, dim=128, page=128, block=128,
             keep=48, query_block=128, sinks=1560, recent=0, causal=False, packed=False, dtype="bf16", ragged=False),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["pack", "read", "packed", "packed", "sparse", "sparse", "sparse"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    dim = rng.choice([64, 128, 128])
    dtype = rng.choice(["bf16", "fp16"])
    ragged = rng.random() < 0.6
    page = rng.choice([8, 16, 24, 32, 64, 128, 200, 1560])
    common = dict(op=op, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, ragged=ragged)
    if op == "pack":
        seqs, new = rng.choice([(rng.randint(1, 200), 1), (rng.randint(1, 24), _log_int(rng, 2, 600)), (rng.randint(1, 3), _log_int(rng, 300, 4680))])
        layout = rng.choice(["interleaved", "halves", "none"])
        return common | dict(seqs=seqs, new=new, history=_log_int(rng, 1, 6000), heads=0 if layout == "none" else heads, layout=layout)
    if op == "read":
        seqs = _log_int(rng, 1, 64)
        return common | dict(seqs=seqs, kv=max(1, min(_log_int(rng, 1, 24000), 46800 * 8 * 128 // (seqs * kv_heads * dim))))
    if op == "packed":
        seqs, new, top = rng.choice([(rng.randint(1, 64), 1, 16384), (rng.randint(1, 16), rng.randint(2, 40), 16384),
                                     (rng.randint(1, 8), _log_int(rng, 40, 1100), 8192), (1, _log_int(rng, 1000, 4680), 23400)])
        kv = new + _log_int(rng, 1, top)
        kv = max(new, min(kv, 1_300_000_000 // (seqs * new * heads), 400_000 // seqs))
        return common | dict(seqs=seqs, new=new, kv=kv, heads=heads, causal=rng.random() < 0.6)
    block, times = rng.choice([(16, 1), (16, 4), (32, 2), (64, 1), (64, 2), (128, 1), (104, 15), (40, 5)])
    seqs, new, query_block = rng.choice([(_log_int(rng, 1, 48), 1, 1), (rng.randint(1, 8), rng.randint(2, 16), 1),
                                         (rng.randint(1, 6), _log_int(rng, 40, 1100), rng.choice([16, 32, 64, 100])),
                                         (1, _log_int(rng, 1000, 4680), rng.choice([64, 128, 256]))])
    causal = new == 1 or rng.random() < 0.7
    case = common | dict(page=block * times, block=block, seqs=seqs, new=new, query_block=query_block, heads=heads, causal=causal,
                         kv=new + max(1, min(_log_int(rng, 200, 50000), 400_000 // seqs)), keep=rng.choice([4, 16, 32]),
                         sinks=rng.choice([0, 4, 64]), recent=rng.choice([0, 64, 200]), packed=rng.random() < 0.4)
    while _items(case) * _width(case) * block * kv_heads * max(dim, query_block * heads // kv_heads) > 600_000_000:
        case["keep"] //= 2
        if case["keep"] < 2:
            case["new"], case["kv"] = case["new"] // 2, case["kv"] - case["new"] // 2
    case["keep"] = max(1, case["keep"])
    return case


def _spread(case, count, most):
    """Lengths of ``count`` sessions up to ``most``: equal, or spread evenly (golden-ratio steps, the first the longest)."""
    if not case["ragged"]:
        return [most] * count
    return [max(1, math.ceil(most * (1.0 - (i * 0.6180339887) % 1.0))) for i in range(count)]


def _lengths(case):
    """New tokens and total lengths (history and new) of every session."""
    if case["op"] == "read":
        return [0] * case["seqs"], _spread(case, case["seqs"], case["kv"])
    new = _spread(case, case["seqs"], case["new"])
    if case["op"] == "pack":
        return new, [case["history"] + n for n in new]
    # the histories run through their spread the other way round, so that a long chunk does not always meet a long history
    old = _spread(case, case["seqs"], case["kv"] - case["new"])[::-1]
    return new, [o + n if case["kv"] > case["new"] else n for o, n in zip(old, new)]


def _items(case):
    """Query blocks that there may be: every token one, or those of the tokens and a rest for each session."""
    new = _lengths(case)[0]
    most = case["seqs"] * -(-max(new) // case["query_block"])
    return sum(new) if case["query_block"] == 1 else min(most, sum(new) // case["query_block"] + case["seqs"])


def _width(case):
    """Blocks that a query block sees at most: those of the sinks, the chosen ones, the recent and its own."""
    new, totals = _lengths(case)
    span = min(case["query_block"], max(new)) if case["causal"] else max(new)
    most = -(-max(totals) // case["page"]) * (case["page"] // case["block"])
    return min(most, -(-case["sinks"] // case["block"]) + case["keep"] + (span + case["recent"] - 2) // case["block"] + 2)


# -- inputs -----------------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _sections(dim):
    pairs = dim // 2
    return (pairs - 2 * (pairs // 3), pairs // 3, pairs // 3)


def _grid_positions(first, count):
    """Frame, row and column of tokens ``first .. first + count`` of a video of GRID frames."""
    at = torch.arange(first, first + count, device=DEVICE, dtype=torch.int32)
    frame = GRID[0] * GRID[1]
    return torch.stack([at // frame, at % frame // GRID[1], at % GRID[1]], dim=1)


def _table(case, g, totals):
    """A block table in which sessions' pages lie in any order, and the number of pages."""
    counts = [-(-n // case["page"]) for n in totals]
    pages = sum(counts) + 3
    order = torch.randperm(pages, device=DEVICE, generator=g).to(torch.int32)
    slot = torch.arange(max(counts), device=DEVICE)
    number = torch.tensor(counts, device=DEVICE)
    index = (number.cumsum(0) - number)[:, None] + slot
    return torch.where(slot < number[:, None], order[index.clamp(max=pages - 1)], -1).to(torch.int32), pages


def _drift(case, g, shape):
    """Rows of K or V: tokens near each other are alike (as in video and text), and their sizes differ."""
    x = torch.randn(shape, device=DEVICE, generator=g)
    if case["op"] == "sparse":
        x += 1.5 * torch.randn(shape[0], -(-shape[1] // 32), *shape[2:], device=DEVICE, generator=g).repeat_interleave(32, dim=1)[:, :shape[1]]
    return x.mul_(torch.exp(0.4 * torch.randn(*shape[:3], 1, device=DEVICE, generator=g)))


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    new, totals = _lengths(case)
    state = {"case": case, "rows": sum(totals), "max_new": max(new)}
    state["table"], pages = _table(case, g, totals)
    state["kv_lens"] = torch.tensor(totals, dtype=torch.int32, device=DEVICE)
    state["cu_q"] = torch.tensor([0] + new, device=DEVICE).cumsum(0).to(torch.int32)
    state["starts"] = torch.tensor([0] + totals, device=DEVICE).cumsum(0).to(torch.int32)
    for name in ("k", "v"):
        rows = _drift(case, g, (pages, case["page"], case["kv_heads"], case["dim"]))
        if case.get("packed", True):
            state[name + "_codes"], scales = _quantise(rows, case["dtype"])
            state[name + "_scales"] = _scale_pages(scales)
        else:
            state[name + "_pages"] = rows.to(dtype)
        if case["op"] == "sparse" and name == "k":  # what earlier steps left: means of whole blocks
            held = _held(state, "k")
            state["means"] = held.unflatten(1, (-1, case["block"])).mean(dim=2).to(dtype)
        del rows
    tokens = sum(new)
    if case["op"] == "pack":
        heads = case["heads"] + 2 * case["kv_heads"]
        fused = torch.randn(tokens, heads, case["dim"], device=DEVICE, generator=g).to(dtype)
        state["q"], state["k"], state["v"] = fused.split([case["heads"], case["kv_heads"], case["kv_heads"]], dim=1)
        state["positions"] = torch.cat([_grid_positions(t - n, n) for n, t in zip(new, totals)])
    elif case["op"] != "read":
        state["q"] = (torch.randn(tokens, case["heads"], case["dim"], device=DEVICE, generator=g) * 0.7).to(dtype)
    return state


# -- the framework's operators ----------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _rope(dim, layout):
    """The rotation that a model keeps."""
    from reelcache_b200.ops.rope import AxisRope
    return AxisRope(dim, _sections(dim), theta=THETA, layout=layout)


def _run_own(state):
    from reelcache_b200.ops import paged
    case, table, kv_lens, cu_q = (state[n] for n in ("case", "table", "kv_lens", "cu_q"))
    if case.get("packed", True):
        k, v = (paged.PackedPages(state[n + "_codes"], state[n + "_scales"]) for n in ("k", "v"))
    else:
        k, v = state["k_pages"], state["v_pages"]
    if case["op"] == "pack":
        got = {n: state[n] for n in ("k_codes", "k_scales", "v_codes", "v_scales")}
        if case["layout"] == "none":
            paged.store(state["k"], state["v"], k, v, table, kv_lens, cu_q)
            return got
        return got | {"q": paged.append(state["q"], state["k"], state["v"], state["positions"], _rope(case["dim"], case["layout"]),
                                        k, v, table, kv_lens, cu_q)}
    if case["op"] == "read":
        k, v = paged.read(k, v, table, state["starts"], state["rows"], dtype=DTYPES[case["dtype"]])
        return {"k": k, "v": v}
    if case["op"] == "packed":
        out, lse = paged.attention(state["q"], k, v, table, kv_lens, cu_q, max_q_len=state["max_new"], causal=case["causal"],
                                   return_lse=True)
        return {"out": out, "lse": lse}
    paged.block_means(k, state["means"], table, kv_lens, cu_q, max_q_len=state["max_new"])
    chosen = paged.select_blocks(state["q"], state["means"], table, kv_lens, cu_q, block=case["block"], keep=case["keep"],
                                 query_block=case["query_block"], max_q_len=state["max_new"], causal=case["causal"],
                                 sinks=case["sinks"], recent=case["recent"])
    out, lse = paged.attention(state["q"], paged.blocks(k, case["block"]), paged.blocks(v, case["block"]), chosen.table,
                               chosen.kv_lens, chosen.cu_q, max_q_len=chosen.max_q_len, causal=case["causal"], return_lse=True)
    return {"out": out, "lse": lse, "blocks": chosen.table, "means": state["means"]}


# -- plain forms ------------------------------------------------------------------------------------------------------

def _quantise(x, kind):
    """Codes and scales [..., 1] of rows in FP32: the smallest power of two that brings a row to 448 and below."""
    top = x.abs().amax(dim=-1, keepdim=True)
    part, power = torch.frexp(top)  # top = part * 2^power, part from 1/2 to 1; 448 = 0.875 * 2^9
    power = torch.where(top > 0, power - 9 + (part > 0.875), LOW[kind]).clamp(LOW[kind], HIGH[kind])
    codes = torch.ldexp(x, -power).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return codes, (power + 127).to(torch.uint8)


def _scale_pages(scales):
    """Scales [pages, page_size, kv_heads, 1] as pages keep them: [kv_heads, pages, page_size]."""
    return scales[..., 0].permute(2, 0, 1).contiguous().view(torch.float8_e8m0fnu)


def _held(state, name):
    """Values in all pages, FP32."""
    if name + "_pages" in state:
        return state[name + "_pages"].float()
    power = state[name + "_scales"].view(torch.uint8).to(torch.int32) - 127
    return torch.ldexp(state[name + "_codes"].float(), power.permute(1, 2, 0)[..., None])


def _turn(x, positions, case):
    parts = []
    for axis, pairs in enumerate(_sections(case["dim"])):
        frequency = THETA ** (-torch.arange(pairs, device=DEVICE, dtype=torch.float32) / pairs)
        parts.append(positions[:, axis, None].float() * frequency)
    angles = torch.cat(parts, dim=1)[:, None, :]
    cos, sin, x = torch.cos(angles), torch.sin(angles), x.float()
    if case["layout"] == "interleaved":
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)


def _tokens(state):
    """Session of every new token and its position there."""
    counts = (state["cu_q"][1:] - state["cu_q"][:-1]).long()
    total = state["positions"].shape[0] if "positions" in state else state["q"].shape[0]
    seq = torch.repeat_interleave(torch.arange(counts.numel(), device=DEVICE), counts, output_size=total)
    place = torch.arange(total, device=DEVICE) - state["cu_q"][:-1].long()[seq]
    return seq, (state["kv_lens"].long() - counts)[seq] + place


def _pack_plain(state):
    case = state["case"]
    seq, at = _tokens(state)
    page, row = state["table"][seq, at // case["page"]].long(), at % case["page"]
    rows = {"k": state["k"].float(), "v": state["v"].float()}
    got = {n: state[n] for n in ("k_codes", "k_scales", "v_codes", "v_scales")}
    if case["layout"] != "none":
        rows["k"] = _turn(state["k"], state["positions"], case)
        got["q"] = _turn(state["q"], state["positions"], case).to(state["q"].dtype)
    for name in ("k", "v"):
        codes, scales = _quantise(rows[name], case["dtype"])
        got[name + "_codes"].view(torch.uint8)[page, row] = codes.view(torch.uint8)
        got[name + "_scales"].view(torch.uint8)[:, page, row] = scales[..., 0].T
    return got


def _read_plain(state):
    case = state["case"]
    counts = state["kv_lens"].long()
    seq = torch.repeat_interleave(torch.arange(case["seqs"], device=DEVICE), counts, output_size=state["rows"])
    at = torch.arange(state["rows"], device=DEVICE) - state["starts"][:-1].long()[seq]
    page, row = state["table"][seq, at // case["page"]].long(), at % case["page"]
    got = {}
    for name in ("k", "v"):
        power = state[name + "_scales"].view(torch.uint8)[:, page, row].T.to(torch.int32) - 127
        got[name] = torch.ldexp(state[name + "_codes"].view(torch.uint8)[page, row].view(torch.float8_e4m3fn).float(),
                                power[..., None]).to(DTYPES[case["dtype"]])
    return got


def _softmax(s, v):
    """Rows of raw scores (minus infinity where nothing is seen) times v, and their log-sum-exp."""
    top = s.amax(dim=-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    s.sub_(top).exp_()
    total = s.sum(dim=-1, keepdim=True)
    return torch.matmul(s, v) / total.clamp(min=1e-30), (top + torch.log(total)).squeeze(-1)


def _attend_plain(state):
    case = state["case"]
    seqs, page, d, kv_heads = case["seqs"], case["page"], case["dim"], case["kv_heads"]
    seq, at = _tokens(state)
    totals = state["kv_lens"].long()
    new = (state["cu_q"][1:] - state["cu_q"][:-1]).long()
    place = at - (totals - new)[seq]
    pages = state["table"].clamp(min=0).long()
    length = pages.shape[1] * page
    k, v = (_held(state, n)[pages].reshape(seqs, length, kv_heads, d) for n in ("k", "v"))
    keys = torch.arange(length, device=DEVICE)
    v = torch.where((keys < totals[:, None])[..., None, None], v, 0.0)
    q = torch.zeros(seqs, state["max_new"], case["heads"], d, device=DEVICE)
    q[seq, place] = state["q"].float()
    q = q.reshape(seqs, -1, kv_heads, case["heads"] // kv_heads, d).permute(0, 2, 3, 1, 4)
    s = torch.matmul(q.reshape(seqs, kv_heads, -1, d), k.permute(0, 2, 3, 1)).div_(math.sqrt(d))
    first = (totals - new)[:, None] + torch.arange(state["max_new"], device=DEVICE)
    last = first if case["causal"] else (totals - 1)[:, None].expand_as(first)
    s.view(*q.shape[:4], length).masked_fill_((keys > last[..., None])[:, None, None], -math.inf)
    out, lse = _softmax(s, v.permute(0, 2, 1, 3))
    out = out.reshape(q.shape).permute(0, 3, 1, 2, 4).reshape(seqs, -1, case["heads"], d)[seq, place]
    lse = lse.reshape(q.shape[:4]).permute(0, 3, 1, 2).reshape(seqs, -1, case["heads"])[seq, place]
    return {"out": out.to(state["q"].dtype), "lse": lse}


def _means_plain(state):
    """Means of the blocks that hold new tokens, over the tokens that they hold, in 64 bits (a choice hangs on them)."""
    case = state["case"]
    block, page = case["block"], case["page"]
    totals = state["kv_lens"].long()
    first = totals - (state["cu_q"][1:] - state["cu_q"][:-1]).long()
    most = state["table"].shape[1] * page // block
    at = torch.arange(most, device=DEVICE)
    touched = (at >= first[:, None] // block) & (at * block < totals[:, None]) & (totals > first)[:, None]
    seq, b = touched.nonzero(as_tuple=True)
    where, part = state["table"][seq, b * block // page].long(), b % (page // block)
    row = part[:, None] * block + torch.arange(block, device=DEVICE)
    if "k_pages" in state:
        keys = state["k_pages"][where[:, None], row].double()
    else:
        power = state["k_scales"].view(torch.uint8)[:, where[:, None], row].permute(1, 2, 0).to(torch.int32) - 127
        keys = torch.ldexp(state["k_codes"].view(torch.uint8)[where[:, None], row].view(torch.float8_e4m3fn).float(), power[..., None]).double()
    there = (totals[seq] - b * block).clamp(max=block)
    keys = torch.where((torch.arange(block, device=DEVICE) < there[:, None])[..., None, None], keys, 0.0)
    state["means"][where, part] = (keys.sum(dim=1) / there[:, None, None]).to(state["means"].dtype)


def _sparse_plain(state):
    case = state["case"]
    _means_plain(state)
    block, d, kv_heads, heads, seqs, each = (case[n] for n in ("block", "dim", "kv_heads", "heads", "seqs", "query_block"))
    group, per_page, q = heads // kv_heads, case["page"] // block, state["q"]
    totals, cu = state["kv_lens"].long(), state["cu_q"].long()
    new = cu[1:] - cu[:-1]
    # query blocks, session by session: session, first new token, tokens
    items, width = _items(case), _width(case)
    number = (new + each - 1) // each
    ends = number.cumsum(0)
    index = torch.arange(items, device=DEVICE)
    seq = torch.searchsorted(ends, index, right=True).clamp(max=seqs - 1)
    start = (index - (ends - number)[seq]) * each
    count = torch.where(index < ends[-1], (new[seq] - start).clamp(max=each), 0)
    first = (totals - new)[seq] + start
    end = torch.where(count > 0, first + count if case["causal"] else totals[seq], 0)
    # scores in 64 bits: values next to a border decide
    token = (cu[seq] + start)[:, None] + torch.arange(each, device=DEVICE)
    there = torch.arange(each, device=DEVICE) < count[:, None]
    rows = torch.where(there[..., None, None], q[token.clamp(max=q.shape[0] - 1)].double(), 0.0)
    blocks = state["table"].shape[1] * per_page
    small = (state["table"].long()[:, :, None] * per_page + torch.arange(per_page, device=DEVICE)).reshape(seqs, blocks)
    means = state["means"].flatten(0, 1)[small.clamp(min=0)].double()  # [seqs, blocks, kv_heads, d]
    pooled = rows.sum(dim=1).reshape(items, kv_heads, group, d)
    most = -(-state["max_new"] // each)
    padded = torch.zeros(seqs, most, kv_heads, group, d, device=DEVICE, dtype=torch.float64)
    live = count > 0
    padded[seq[live], (start // each)[live]] = pooled[live]
    score = torch.matmul(padded.permute(0, 2, 1, 3, 4).reshape(seqs, kv_heads, most * group, d), means.permute(0, 2, 3, 1))
    score = score.reshape(seqs, kv_heads, most, group, blocks).amax(dim=3)[seq, :, (start // each).clamp(max=most - 1)]  # [items, kv_heads, blocks]
    # always: the sinks' blocks, the recent ones and the new tokens' own
    at = torch.arange(blocks, device=DEVICE)
    seen = (at * block < end[:, None])
    near = ((first if case["causal"] else (totals - new)[seq]) - case["recent"]).clamp(min=0)
    always = seen & ((at < -(-case["sinks"] // block)) | (at >= near[:, None] // block))
    free = (seen & ~always)[:, None].expand_as(score)
    score = torch.where(free, score, -math.inf)
    rank = torch.argsort(torch.argsort(score, dim=-1, descending=True, stable=True), dim=-1)
    taken = (free & (rank < case["keep"])) | always[:, None]
    order = torch.sort(torch.where(taken, at, blocks), dim=-1).values[..., :width]  # the chosen blocks, in order
    real = order < blocks
    pages = torch.where(real, small[seq][:, None].expand(-1, kv_heads, -1).gather(-1, order.clamp(max=blocks - 1)), -1)
    # attention over them
    place = order[..., None] * block + torch.arange(block, device=DEVICE)
    row = pages.clamp(min=0)[..., None] * block + torch.arange(block, device=DEVICE)
    row, place = row.flatten(-2), torch.where(real[..., None], place, 1 << 30).flatten(-2)
    head = torch.arange(kv_heads, device=DEVICE)[:, None]
    if case["packed"]:
        k, v = (torch.ldexp(state[n + "_codes"].view(torch.uint8).flatten(0, 1)[row, head].view(torch.float8_e4m3fn).float(),
                            (state[n + "_scales"].view(torch.uint8).flatten(1)[head, row].to(torch.int32) - 127)[..., None]) for n in ("k", "v"))
    else:
        k, v = (state[n + "_pages"].flatten(0, 1)[row, head].float() for n in ("k", "v"))
    v = torch.where((place < end[:, None, None])[..., None], v, 0.0)
    x = rows.float().reshape(items, each, kv_heads, group, d).permute(0, 2, 1, 3, 4).reshape(items, kv_heads, each * group, d)
    s = torch.matmul(x, k.transpose(-1, -2)).div_(math.sqrt(d))
    last = first[:, None] + torch.arange(each, device=DEVICE) if case["causal"] else (end - 1)[:, None].expand(-1, each)
    last = last.repeat_interleave(group, dim=1)
    s.masked_fill_(place[:, :, None] > last[:, None, :, None], -math.inf)
    out, lse = _softmax(s, v)
    out = out.reshape(items, kv_heads, each, group, d).permute(0, 2, 1, 3, 4).reshape(items, each, heads, d)
    lse = lse.reshape(items, kv_heads, each, group).permute(0, 2, 1, 3).reshape(items, each, heads)
    got = {"out": torch.empty_like(q), "lse": torch.empty(q.shape[:2], device=DEVICE)}
    got["out"][token[there]] = out[there].to(q.dtype)
    got["lse"][token[there]] = lse[there]
    return got | {"blocks": pages.to(torch.int32), "means": state["means"]}


def run(state):
    if own:
        return _run_own(state)
    return {"pack": _pack_plain, "read": _read_plain, "packed": _attend_plain, "sparse": _sparse_plain}[state["case"]["op"]](state)


# -- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    new, totals = _lengths(case)
    d, kv_heads, tokens = case["dim"], case["kv_heads"], sum(new)
    packed_row = 2 * kv_heads * (d + 1)  # K and V of a token
    if case["op"] == "pack":
        turned = case["heads"] + kv_heads if case["heads"] else 0
        return {"bytes": tokens * (2 * (2 * case["heads"] + 2 * kv_heads) * d + packed_row + (12 if turned else 0)),
                "flops": tokens * d * (3 * turned + 4 * kv_heads)}
    if case["op"] == "read":
        return {"bytes": sum(totals) * (packed_row + 4 * kv_heads * d), "flops": sum(totals) * 2 * kv_heads * d}
    heads = case["heads"]
    rows = tokens * heads * (4 * d + 4)  # q, out and lse
    if case["op"] == "packed":
        pairs = sum(n * t - (n * (n - 1) // 2 if case["causal"] else 0) for n, t in zip(new, totals))
        return {"bytes": rows + sum(totals) * packed_row, "flops": 4 * pairs * heads * d}
    block, each = case["block"], case["query_block"]
    pairs = seen = scored = touched = 0
    for n, total in zip(new, totals):
        touched += n + (total - n) % block
        whole = 0
        for start in range(0, n, each):
            count = min(each, n - start)
            first = total - n + start
            end = first + count if case["causal"] else total
            near = max(0, (first if case["causal"] else total - n) - case["recent"])
            blocks = -(-end // block)
            always = blocks - near // block + min(-(-case["sinks"] // block), near // block)
            chosen = min(case["keep"], blocks - always)
            keys = end - (blocks - always - chosen) * block
            pairs += count * keys - (count * (count - 1) // 2 if case["causal"] else 0)
            whole += keys
            scored += blocks
        seen += min(whole, total)
    held = packed_row if case["packed"] else 4 * kv_heads * d
    means = 2 * kv_heads * d * (sum(-(-t // block) for t in totals) + -(-touched // block))
    return {"bytes": rows + seen * held + touched * held // 2 + means, "flops": 4 * pairs * heads * d + 2 * scored * heads * d}


# -- the definitions in 64 bits ---------------------------------------------------------------------------------------

def _spun(x, positions, case):
    """Pairs as complex numbers times e^(i angle), in 64 bits."""
    angle = torch.cat([positions[:, a:a + 1].double() / THETA ** (torch.arange(n, device=DEVICE, dtype=torch.float64) / n)
                       for a, n in enumerate(_sections(case["dim"]))], dim=1)
    factor = torch.polar(torch.ones_like(angle), angle)[:, None, :]
    x = x.double()
    if case["layout"] == "interleaved":
        return torch.view_as_real(torch.view_as_complex(x.reshape(*x.shape[:-1], -1, 2).contiguous()) * factor).reshape(x.shape)
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * factor
    return torch.cat([z.real, z.imag], dim=-1)


def _nearest(x, kind):
    """Values of codes and scales of rows in 64 bits: four significant bits, in steps of 2^-9 at least."""
    top = x.abs().amax(dim=-1, keepdim=True)
    power = torch.ceil(torch.log2(top.clamp(min=1e-300) / 448.0) - 1e-13).clamp(LOW[kind], HIGH[kind])
    x = (x * torch.exp2(-power)).clamp(-448.0, 448.0)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3.0)
    return torch.round(x / step) * step, torch.exp2(power[..., 0])


def _values(state, name):
    """Values in all pages, 64 bits."""
    if name + "_pages" in state:
        return state[name + "_pages"].double()
    return state[name + "_codes"].double() * state[name + "_scales"].double().permute(1, 2, 0)[..., None]


def exact(case, seed):
    state = prepare(case, seed)
    new, totals = _lengths(case)
    group = case["heads"] // case["kv_heads"] if case.get("heads") else 1
    if case["op"] == "pack":
        got = {n: state[n].double() for n in ("k_codes", "k_scales", "v_codes", "v_scales")}
        rows = {"k": state["k"].double(), "v": state["v"].double()}
        if case["layout"] != "none":
            rows["k"], got["q"] = (_spun(state[n], state["positions"], case) for n in ("k", "q"))
        first = 0
        for s, (n, total) in enumerate(zip(new, totals)):
            at = torch.arange(total - n, total, device=DEVICE)
            page, row = state["table"][s].long()[at // case["page"]], at % case["page"]
            for name in ("k", "v"):
                codes, scales = _nearest(rows[name][first:first + n], case["dtype"])
                got[name + "_codes"][page, row] = codes
                got[name + "_scales"][:, page, row] = scales.T
            first += n
        return got
    if case["op"] == "read":
        k, v = (torch.cat([_values(state, m)[state["table"][s][:-(-t // case["page"])].long()].flatten(0, 1)[:t]
                           for s, t in enumerate(totals)]) for m in ("k", "v"))
        return {"k": k, "v": v}
    values = {m: _values(state, m) for m in ("k", "v")}
    out, lse = torch.empty(state["q"].shape, dtype=torch.float64, device=DEVICE), torch.empty(state["q"].shape[:2], dtype=torch.float64, device=DEVICE)
    means, first = state["means"].double() if case["op"] == "sparse" else None, 0
    for s, (n, total) in enumerate(zip(new, totals)):
        held = state["table"][s][:-(-total // case["page"])].long()
        k, v = (values[m][held].flatten(0, 1)[:total] for m in ("k", "v"))
        q, at = state["q"][first:first + n].double(), torch.arange(total, device=DEVICE)
        last = torch.arange(total - n, total, device=DEVICE)[:, None] if case["causal"] else torch.full((n, 1), total - 1, device=DEVICE)
        seen = (at <= last).expand(case["kv_heads"], -1, -1)
        if case["op"] == "sparse":
            block = case["block"]
            blocks = -(-total // block)
            per_page = case["page"] // block
            for b in range((total - n) // block, blocks):
                means[held[b // per_page], b % per_page] = k[b * block:(b + 1) * block].mean(dim=0)
            m = means[held].flatten(0, 1)[:blocks].to(state["means"].dtype).double()
            seen = seen.clone()
            for start in range(0, n, case["query_block"]):
                rows = slice(start, min(n, start + case["query_block"]))
                end = total - n + rows.stop if case["causal"] else total
                near = max(0, total - n + (start if case["causal"] else 0) - case["recent"])
                there = -(-end // block)
                score = torch.einsum("hgd,bhd->hgb", q[rows].sum(dim=0).unflatten(0, (-1, group)), m[:there]).amax(dim=1)
                low, high = min(-(-case["sinks"] // block), near // block), near // block
                kept = torch.ones_like(score, dtype=torch.bool)
                kept[:, low:high] = False
                best = torch.sort(score[:, low:high], dim=1, descending=True, stable=True).indices[:, :case["keep"]] + low
                kept.scatter_(1, best, True)
                seen[:, rows] &= kept.repeat_interleave(block, dim=1)[:, None, :total] if there == blocks else \
                    torch.nn.functional.pad(kept, (0, blocks - there)).repeat_interleave(block, dim=1)[:, None, :total]
        for h in range(case["heads"]):
            score = (q[:, h] @ k[:, h // group].T) * case["dim"] ** -0.5
            score = torch.where(seen[h // group], score, -math.inf)
            lse[first:first + n, h] = torch.logsumexp(score, dim=1)
            out[first:first + n, h] = torch.exp(score - lse[first:first + n, h, None]) @ v[:, h // group]
        first += n
    return {"out": out, "lse": lse} if case["op"] == "packed" else {"out": out, "lse": lse, "blocks": None, "means": means}
