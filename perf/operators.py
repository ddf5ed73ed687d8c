"""What the paged-cache operators are measured on: cases over their range of use, their plain forms and 64-bit values.

Four operators, each a part of one path (a session's new tokens are rotated, written into its pages, attended with its
history, and its pages are shared, grown, freed and moved):

``rotate``   rotary positions of several axes (frame, row, column) on q and k, with the gradient
``append``   the same rotation on the way into a paged cache: q rotated, k rotated into pages, v copied into pages
``attend``   attention of new tokens over the paged cache, single tokens and chunks, with its log-sum-exp
``pages``    the page table: forked sessions share their history's pages and grow, finished ones are freed and the
             pages compacted
"""

import functools
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
THETA = 10000.0
GRID = (30, 52)  # latent rows and columns of a frame: 1,560 tokens


# -- cases ------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # training on one latent frame of a 12-head video model
        dict(name="rotate_frame", op="rotate", tokens=1560, heads=12, kv_heads=12, dim=128, layout="interleaved", dtype="bf16"),
        # training on a text-and-image sample of a small grouped-head model kept in 32 bits, odd length
        dict(name="rotate_grouped", op="rotate", tokens=4097, heads=16, kv_heads=4, dim=64, layout="halves", dtype="fp32"),
        # training on four 720p latent frames with 32 heads
        dict(name="rotate_video", op="rotate", tokens=14400, heads=32, kv_heads=32, dim=128, layout="interleaved", dtype="bf16"),
        # one decoding step of 61 sessions: a token each into pages of 16
        dict(name="append_step", op="append", seqs=61, new=1, history=4096, heads=32, kv_heads=8, dim=128, page=16,
             layout="halves", dtype="fp16", ragged=False),
        # a chunk of three latent frames for each of three sessions, one frame to a page
        dict(name="append_chunk", op="append", seqs=3, new=4680, history=9360, heads=12, kv_heads=12, dim=128, page=1560,
             layout="interleaved", dtype="bf16", ragged=False),
        # one token of one session: latency
        dict(name="attend_token", op="attend", seqs=1, new=1, kv=2048, heads=32, kv_heads=8, dim=128, page=16, causal=True,
             window=0, sinks=0, dtype="bf16", ragged=False),
        # a decoding step of 48 sessions of very different lengths
        dict(name="attend_step", op="attend", seqs=48, new=1, kv=16384, heads=32, kv_heads=8, dim=128, page=64, causal=True,
             window=0, sinks=0, dtype="bf16", ragged=True),
        # pieces of prompts of eight sessions, each a different length, after histories of different lengths
        dict(name="attend_prompts", op="attend", seqs=8, new=1021, kv=8192, heads=32, kv_heads=8, dim=128, page=32, causal=True,
             window=0, sinks=0, dtype="fp16", ragged=True),
        # a chunk of three latent frames that sees itself and four chunks before it
        dict(name="attend_chunk", op="attend", seqs=1, new=4680, kv=23400, heads=12, kv_heads=12, dim=128, page=1560,
             causal=False, window=0, sinks=0, dtype="bf16", ragged=False),
        # a chunk late in a long session: a window of 21 latent frames and a sink chunk, a quarter of 40 heads
        dict(name="attend_window", op="attend", seqs=1, new=4680, kv=46800, heads=10, kv_heads=10, dim=128, page=1560,
             causal=False, window=32760, sinks=4680, dtype="bf16", ragged=False),
        # sessions forked inside a page, then grown: shared history, copied tails, new pages
        dict(name="pages_fork", op="pages", kind="fork", pages=2048, page=16, planes=48, width=512, seqs=96, count=37, length=700,
             dtype="bf16"),
        # finished sessions freed, the pages of the rest moved together
        dict(name="pages_compact", op="pages", kind="compact", pages=1536, page=64, planes=24, width=512, seqs=64, count=29,
             length=1500, dtype="bf16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotate", "append", "attend", "attend", "attend", "pages"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    dim = rng.choice([64, 128, 128])
    if op == "rotate":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        tokens = min(_log_int(rng, 1, 20000), int(14400 * 64 * 128 * 2 / ((heads + kv_heads) * dim * (4 if dtype == "fp32" else 2))))
        return dict(op=op, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim,
                    layout=rng.choice(["interleaved", "halves"]), dtype=dtype)
    page = rng.choice([8, 16, 24, 32, 64, 128, 200, 1560])
    if op == "append":
        seqs, new = rng.choice([(rng.randint(1, 200), 1), (rng.randint(1, 24), _log_int(rng, 2, 600)), (rng.randint(1, 3), _log_int(rng, 300, 4680))])
        return dict(op=op, seqs=seqs, new=new, history=_log_int(rng, 1, 6000), heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                    layout=rng.choice(["interleaved", "halves"]), dtype=rng.choice(["bf16", "fp16"]), ragged=rng.random() < 0.5)
    if op == "attend":
        seqs, new, top = rng.choice([(rng.randint(1, 64), 1, 16384), (rng.randint(1, 16), rng.randint(2, 40), 16384),
                                     (rng.randint(1, 8), _log_int(rng, 40, 1100), 8192), (1, _log_int(rng, 1000, 4680), 30000)])
        kv = new + _log_int(rng, 1, top)
        kv = max(new, min(kv, 1_750_000_000 // (seqs * new * heads), 400_000 // seqs))
        windowed = rng.random() < 0.3
        window = _log_int(rng, 16, max(17, kv)) if windowed else 0
        return dict(op=op, seqs=seqs, new=new, kv=kv, heads=heads, kv_heads=kv_heads, dim=dim, page=page, causal=rng.random() < 0.6,
                    window=window, sinks=rng.choice([0, 4, 100, 1560]) if windowed else 0, dtype=rng.choice(["bf16", "fp16"]), ragged=rng.random() < 0.6)
    page = rng.choice([8, 16, 32, 64])
    planes = rng.choice([2, 16, 48])
    width = rng.choice([128, 512])
    pages = min(_log_int(rng, 64, 4096), 2048 * 16 * 48 * 512 // (page * planes * width))
    seqs = min(rng.randint(8, 128), pages // 6)
    length = min(_log_int(rng, page // 2, 40 * page), max(1, page * (pages // (2 * seqs))))
    return dict(op=op, kind=rng.choice(["fork", "compact"]), pages=pages, page=page, planes=planes, width=width, seqs=seqs,
                count=rng.randint(1, seqs // 2), length=length, dtype=rng.choice(["bf16", "fp16"]))


def _spread(case, count, most):
    """Lengths of ``count`` sessions up to ``most``: equal, or spread evenly (golden-ratio steps, the first the longest)."""
    if not case.get("ragged"):
        return [most] * count
    return [max(1, math.ceil(most * (1.0 - (i * 0.6180339887) % 1.0))) for i in range(count)]


def _lengths(case):
    """New tokens and total lengths (history and new) of every session."""
    new = _spread(case, case["seqs"], case["new"])
    if case["op"] == "append":
        return new, [case["history"] + n for n in new]
    # the histories run through their spread the other way round, so that a long chunk does not always meet a long history
    old = _spread(case, case["seqs"], case["kv"] - case["new"])[::-1]
    return new, [o + n if case["kv"] > case["new"] else n for o, n in zip(old, new)]


def _fork_plan(case):
    """Sessions' lengths, and the parent, child and length of each fork (children are sessions without pages). In a fork
    case the first half of the sessions have pages; a compaction case uses them all."""
    seqs, page = case["seqs"], case["page"]
    live = seqs // 2 if case["kind"] == "fork" else seqs
    lens = [max(1, math.ceil(case["length"] * (1.0 - (i * 0.6180339887) % 1.0))) for i in range(live)] + [0] * (seqs - live)
    while sum(-(-n // page) for n in lens) > case["pages"] - 4 * case["count"]:  # a child takes three new pages at most
        lens = [n // 2 for n in lens]
    parents = [(i * 7) % live for i in range(case["count"])]
    children = [live + i for i in range(case["count"])]
    at = [lens[p] - (i % 3) * (lens[p] // 4) for i, p in enumerate(parents)]
    grown = [n + 1 + (i * 11) % (2 * page) for i, n in enumerate(at)]
    return lens, parents, children, at, grown


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


def _paged(case, g, totals):
    """K and V pages with a table in which sessions' pages lie in any order; what no session holds is old data."""
    page = case["page"]
    counts = [-(-n // page) for n in totals]
    width = max(counts)
    pages = sum(counts) + 3
    dtype = DTYPES[case["dtype"]]
    k = (torch.randn(pages, page, case["kv_heads"], case["dim"], device=DEVICE, generator=g) * 1.5).to(dtype)
    v = torch.randn(pages, page, case["kv_heads"], case["dim"], device=DEVICE, generator=g).to(dtype)
    order = torch.randperm(pages, device=DEVICE, generator=g).to(torch.int32)
    slot = torch.arange(width, device=DEVICE)
    number = torch.tensor(counts, device=DEVICE)
    index = (number.cumsum(0) - number)[:, None] + slot
    table = torch.where(slot < number[:, None], order[index.clamp(max=pages - 1)], -1).to(torch.int32)
    return k, v, table


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "rotate":
        n, d = case["tokens"], case["dim"]
        for name, heads in (("q", case["heads"]), ("k", case["kv_heads"])):
            state[name] = torch.randn(n, heads, d, device=DEVICE, generator=g).to(dtype).requires_grad_()
            state["d" + name] = torch.randn(n, heads, d, device=DEVICE, generator=g).to(dtype)
        state["positions"] = _grid_positions(4680 * (seed % 5), n)
        return state
    if case["op"] == "pages":
        lens, parents, children, at, grown = _fork_plan(case)
        counts = torch.tensor([-(-n // case["page"]) for n in lens], device=DEVICE)
        width = int(counts.max()) + 3
        order = torch.randperm(case["pages"], device=DEVICE, generator=g).to(torch.int32)
        slot = torch.arange(width, device=DEVICE)
        index = (counts.cumsum(0) - counts)[:, None] + slot
        held = slot < counts[:, None]
        table = torch.where(held, order[index.clamp(max=case["pages"] - 1)], -1).to(torch.int32)
        refs = torch.zeros(case["pages"], dtype=torch.int32, device=DEVICE)
        refs[table[held].long()] = 1
        if case["kind"] == "compact":  # some sessions hold their first page in common with the one before
            shared = torch.arange(1, case["seqs"], 4, device=DEVICE)
            shared = shared[(counts[shared] > 1) & (counts[shared - 1] > 1)]
            refs[table[shared, 0].long()] = 0
            table[shared, 0] = table[shared - 1, 0]
            refs[table[shared, 0].long()] = 2
        lens = torch.tensor(lens, dtype=torch.int32, device=DEVICE)
        state["packed"] = torch.cat([refs, lens, table.reshape(-1)])
        state["width"] = width
        state["storage"] = torch.randn(case["planes"], case["pages"], case["page"], case["width"], device=DEVICE, generator=g, dtype=dtype)
        if case["kind"] == "fork":
            for name, value in (("parents", parents), ("children", children), ("at", at), ("grown", grown)):
                state[name] = torch.tensor(value, dtype=torch.int32, device=DEVICE)
        else:
            done = torch.randperm(case["seqs"], device=DEVICE, generator=g)[:case["count"]]
            state["done"] = done.sort().values.to(torch.int32)
        return state
    new, totals = _lengths(case)
    state["k_pages"], state["v_pages"], state["table"] = _paged(case, g, totals)
    state["kv_lens"] = torch.tensor(totals, dtype=torch.int32, device=DEVICE)
    state["cu_q"] = torch.tensor([0] + new, device=DEVICE).cumsum(0).to(torch.int32)
    state["max_new"] = max(new)
    tokens = sum(new)
    if case["op"] == "append":
        heads = case["heads"] + 2 * case["kv_heads"]
        fused = torch.randn(tokens, heads, case["dim"], device=DEVICE, generator=g).to(dtype)
        state["q"], state["k"], state["v"] = fused.split([case["heads"], case["kv_heads"], case["kv_heads"]], dim=1)
        state["positions"] = torch.cat([_grid_positions(t - n, n) for n, t in zip(new, totals)])
    else:
        state["q"] = (torch.randn(tokens, case["heads"], case["dim"], device=DEVICE, generator=g) * 1.5).to(dtype)
    return state


# -- the framework's operators ----------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _rope(dim, layout):
    """The rotation that a model keeps."""
    from reelcache_b200.ops.rope import AxisRope
    return AxisRope(dim, _sections(dim), theta=THETA, layout=layout)


def _run_own(state):
    from reelcache_b200.ops import paged, rope
    case = state["case"]
    if case["op"] == "rotate":
        q, k = rope.rotate(state["q"], state["k"], state["positions"], _rope(case["dim"], case["layout"]))
        dq, dk = torch.autograd.grad((q, k), (state["q"], state["k"]), (state["dq"], state["dk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if case["op"] == "append":
        q = paged.append(state["q"], state["k"], state["v"], state["positions"], _rope(case["dim"], case["layout"]),
                         state["k_pages"], state["v_pages"], state["table"], state["kv_lens"], state["cu_q"])
        return {"q": q, "k_pages": state["k_pages"], "v_pages": state["v_pages"]}
    if case["op"] == "attend":
        out, lse = paged.attention(state["q"], state["k_pages"], state["v_pages"], state["table"], state["kv_lens"], state["cu_q"],
                                   max_q_len=state["max_new"], causal=case["causal"], window=case["window"] or None,
                                   sinks=case["sinks"], return_lse=True)
        return {"out": out, "lse": lse}
    table = paged.PageTable(state["packed"].clone(), pages=case["pages"], seqs=case["seqs"], page_size=case["page"])
    if case["kind"] == "fork":
        table.fork(state["parents"], state["children"], state["at"], state["storage"])
        table.allocate(state["children"], state["grown"])
    else:
        table.release(state["done"])
        table.compact(state["storage"])
    return {"refcount": table.refcount, "lens": table.lens, "table": table.block_table, "storage": state["storage"]}


# -- plain forms ------------------------------------------------------------------------------------------------------

def _angles(case, positions):
    parts = []
    for axis, pairs in enumerate(_sections(case["dim"])):
        frequency = THETA ** (-torch.arange(pairs, device=DEVICE, dtype=torch.float32) / pairs)
        parts.append(positions[:, axis, None].float() * frequency)
    angles = torch.cat(parts, dim=1)[:, None, :]
    return torch.cos(angles), torch.sin(angles)


def _turn(x, cos, sin, layout):
    x = x.float()
    if layout == "interleaved":
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)


def _visible(case, place, total, keys):
    """Which of the positions ``keys`` the query at position ``place`` of a session of ``total`` tokens sees."""
    last = place if case["causal"] else total - 1
    seen = keys <= last
    if case["window"]:
        seen = seen & ((keys > last - case["window"]) | (keys < case["sinks"]))
    return seen


def _tokens(state):
    """Session and place in the session's new tokens of every token."""
    counts = (state["cu_q"][1:] - state["cu_q"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(counts.numel(), device=DEVICE), counts, output_size=state["q"].shape[0])
    return seq, torch.arange(state["q"].shape[0], device=DEVICE) - state["cu_q"][:-1].long()[seq], counts


def _attend_plain(state):
    case = state["case"]
    seqs, page, d = case["seqs"], case["page"], case["dim"]
    groups = case["heads"] // case["kv_heads"]
    seq, place, counts = _tokens(state)
    totals = state["kv_lens"].long()
    pages = state["table"].clamp(min=0).long()
    length = pages.shape[1] * page
    k = state["k_pages"][pages].reshape(seqs, length, case["kv_heads"], d).float()
    v = state["v_pages"][pages].reshape(seqs, length, case["kv_heads"], d).float()
    keys = torch.arange(length, device=DEVICE)
    v = torch.where((keys < totals[:, None])[..., None, None], v, 0.0)
    q = torch.zeros(seqs, state["max_new"], case["heads"], d, device=DEVICE)
    q[seq, place] = state["q"].float()
    q = q.reshape(seqs, -1, case["kv_heads"], groups, d).permute(0, 2, 3, 1, 4).reshape(seqs, case["kv_heads"], -1, d)
    s = torch.matmul(q, k.permute(0, 2, 3, 1)) / math.sqrt(d)
    s = s.reshape(seqs, case["kv_heads"], groups, state["max_new"], length)
    at = (totals - counts)[:, None] + torch.arange(state["max_new"], device=DEVICE)
    seen = _visible(case, at[..., None], totals[:, None, None], keys)
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(dim=-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    s.sub_(top).exp_()
    total = s.sum(dim=-1, keepdim=True)
    out = torch.matmul(s.reshape(seqs, case["kv_heads"], -1, length), v.permute(0, 2, 1, 3))
    out = out.reshape(seqs, case["kv_heads"], groups, -1, d) / total.clamp(min=1e-30)
    lse = (top + torch.log(total)).squeeze(-1)
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs, -1, case["heads"], d)[seq, place]
    lse = lse.permute(0, 3, 1, 2).reshape(seqs, -1, case["heads"])[seq, place]
    return {"out": out.to(state["q"].dtype), "lse": lse}


def _pages_plain(state):
    case = state["case"]
    pages, seqs, page, storage = case["pages"], case["seqs"], case["page"], state["storage"]
    packed = state["packed"].clone()
    refs, lens, table = packed[:pages], packed[pages:pages + seqs], packed[pages + seqs:].view(seqs, -1)
    slot = torch.arange(table.shape[1], device=DEVICE)
    if case["kind"] == "fork":
        parents, children, at = (state[n].long() for n in ("parents", "children", "at"))
        free = torch.argsort((refs != 0).int(), stable=True)  # free pages first, the lowest first
        full = at // page
        part = at % page > 0
        shared = slot < full[:, None]
        rows = torch.where(shared, table[parents], -1)
        refs.index_add_(0, rows[shared].long(), torch.ones_like(rows[shared]))
        tails = free[part.cumsum(0) - 1]
        source = table[parents, full.clamp(max=table.shape[1] - 1)].long()
        rows = torch.where((slot == full[:, None]) & part[:, None], tails[:, None], rows).to(torch.int32)
        refs[tails[part]] = 1
        table[children] = rows
        lens[children] = at.to(torch.int32)
        kept = torch.arange(page, device=DEVICE) < (at % page)[part][:, None]
        storage[:, tails[part]] = torch.where(kept[None, :, :, None], storage[:, source[part]], storage[:, tails[part]])
        grown = state["grown"].long()
        free = torch.argsort((refs != 0).int(), stable=True)
        fresh = (slot >= (-(-at // page))[:, None]) & (slot < (-(-grown // page))[:, None])
        order = fresh.reshape(-1).cumsum(0).reshape(fresh.shape) - 1
        rows = torch.where(fresh, free[order.clamp(min=0)], rows).to(torch.int32)
        refs[rows[fresh].long()] = 1
        table[children] = rows
        lens[children] = grown.to(torch.int32)
    else:
        done = state["done"].long()
        rows = table[done]
        refs.index_add_(0, rows[rows >= 0].long(), -torch.ones_like(rows[rows >= 0]))
        table[done] = -1
        lens[done] = 0
        live = refs != 0
        count = live.sum()
        index = torch.arange(pages, device=DEVICE)
        source = index[live & (index >= count)]
        target = index[~live & (index < count)]
        storage[:, target] = storage[:, source]
        place = index.clone()
        place[source] = target
        table.copy_(torch.where(table >= 0, place[table.clamp(min=0).long()], -1))
        refs[target] = refs[source]
        refs[source] = 0
    return {"refcount": refs, "lens": lens, "table": table, "storage": storage}


def _run_plain(state):
    case = state["case"]
    if case["op"] == "rotate":
        cos, sin = _angles(case, state["positions"])
        got = {n: _turn(state[n].detach(), cos, sin, case["layout"]) for n in ("q", "k")}
        got |= {n: _turn(state[n], cos, -sin, case["layout"]) for n in ("dq", "dk")}
        return {n: x.to(state["q"].dtype) for n, x in got.items()}
    if case["op"] == "append":
        cos, sin = _angles(case, state["positions"])
        q, k = (_turn(state[n], cos, sin, case["layout"]).to(state["q"].dtype) for n in ("q", "k"))
        seq, place, counts = _tokens(state)
        at = (state["kv_lens"].long() - counts)[seq] + place
        page = state["table"][seq, at // case["page"]].long()
        state["k_pages"][page, at % case["page"]] = k
        state["v_pages"][page, at % case["page"]] = state["v"]
        return {"q": q, "k_pages": state["k_pages"], "v_pages": state["v_pages"]}
    return _attend_plain(state) if case["op"] == "attend" else _pages_plain(state)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# -- what a pass cannot do without ------------------------------------------------------------------------------------

def _pairs(case):
    """(query, key) pairs that are seen and keys that any query sees, over the sessions, for one head."""
    pairs = seen = 0
    for n, total in zip(*_lengths(case)):
        lasts = range(total - n, total) if case["causal"] else [total - 1]
        repeat = 1 if case["causal"] else n
        for last in lasts:
            window = case["window"] or last + 1
            low = max(0, last - window + 1)
            pairs += repeat * (last + 1 - low + min(case["sinks"], low))
        low = max(0, (lasts[0] + 1) - (case["window"] or total + 1))
        seen += total - low + min(case["sinks"], low)
    return pairs, seen


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rotate":
        numbers = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 4 * size * numbers + 12 * case["tokens"], "flops": 2 * 3 * numbers}
    if case["op"] == "pages":
        lens, parents, children, at, grown = _fork_plan(case)
        row = case["planes"] * case["width"] * size
        if case["kind"] == "fork":
            rows = sum(n % case["page"] for n in at)
            table = sum(2 * (n // case["page"]) for n in at) + sum(-(-n // case["page"]) for n in grown)
        else:  # the freed sessions are drawn by seed: on average this share of the pages stays, and of those this one moves
            held = sum(-(-n // case["page"]) for n in lens)
            stay = held * (case["seqs"] - case["count"]) / case["seqs"]
            rows = case["page"] * stay * (1 - stay / case["pages"])
            table = 2 * held
        return {"bytes": int(2 * rows * row + 4 * (table + case["pages"])), "flops": 0}
    new = sum(_lengths(case)[0])
    q = new * case["heads"] * case["dim"] * size
    if case["op"] == "append":
        kv = new * 2 * case["kv_heads"] * case["dim"] * size
        return {"bytes": 2 * (q + kv) + 12 * new, "flops": 3 * new * (case["heads"] + case["kv_heads"]) * case["dim"]}
    pairs, seen = _pairs(case)
    kv = 2 * seen * case["kv_heads"] * case["dim"] * size
    return {"bytes": 2 * q + kv + 4 * new * case["heads"], "flops": 4 * pairs * case["heads"] * case["dim"]}


# -- the definitions in 64 bits ---------------------------------------------------------------------------------------

def _spun(x, positions, case, sign=1.0):
    """Pairs as complex numbers times e^(i angle), in 64 bits."""
    angle = torch.cat([positions[:, a:a + 1].double() / THETA ** (torch.arange(n, device=DEVICE, dtype=torch.float64) / n)
                       for a, n in enumerate(_sections(case["dim"]))], dim=1)
    factor = torch.polar(torch.ones_like(angle), sign * angle)[:, None, :]
    x = x.detach().double()
    if case["layout"] == "interleaved":
        return torch.view_as_real(torch.view_as_complex(x.reshape(*x.shape[:-1], -1, 2).contiguous()) * factor).reshape(x.shape)
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * factor
    return torch.cat([z.real, z.imag], dim=-1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotate":
        return {n: _spun(state[n], state["positions"], case, -1.0 if n[0] == "d" else 1.0) for n in ("q", "k", "dq", "dk")}
    if case["op"] == "pages":
        return None  # whole numbers and moved values: nothing is computed
    new, totals = _lengths(case)
    if case["op"] == "append":
        pages = {n: state[n + "_pages"].double() for n in ("k", "v")}
        turned = {"k": _spun(state["k"], state["positions"], case), "v": state["v"].double()}
        first = 0
        for s, (n, total) in enumerate(zip(new, totals)):
            at = torch.arange(total - n, total, device=DEVICE)
            page = state["table"][s].long()[torch.div(at, case["page"], rounding_mode="floor")]
            for name in pages:
                pages[name][page, at % case["page"]] = turned[name][first:first + n]
            first += n
        return {"q": _spun(state["q"], state["positions"], case), "k_pages": pages["k"], "v_pages": pages["v"]}
    groups = case["heads"] // case["kv_heads"]
    outs, sums, first = [], [], 0
    for s, (n, total) in enumerate(zip(new, totals)):
        held = state["table"][s][:-(-total // case["page"])].long()
        k, v = (state[m][held].flatten(0, 1)[:total].double() for m in ("k_pages", "v_pages"))
        q = state["q"][first:first + n].double()
        seen = _visible(case, torch.arange(total - n, total, device=DEVICE)[:, None], total, torch.arange(total, device=DEVICE))
        out, lse = torch.empty_like(q), torch.empty(q.shape[:2], dtype=torch.float64, device=DEVICE)
        for h in range(case["heads"]):
            score = (q[:, h] @ k[:, h // groups].T) * case["dim"] ** -0.5
            score = torch.where(seen, score, -math.inf)
            lse[:, h] = torch.logsumexp(score, dim=1)
            out[:, h] = torch.exp(score - lse[:, h, None]).nan_to_num(0.0) @ v[:, h // groups]
        outs.append(out)
        sums.append(lse)
        first += n
    return {"out": torch.cat(outs), "lse": torch.cat(sums)}
