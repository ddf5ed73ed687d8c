"""Plain 64-bit forms of the paged-cache operators, and a page table kept in Python lists."""

import math

import torch


def spun(x, positions, sections, theta, layout, sign=1.0):
    """Rotation by ``sign * phi`` in 64 bits: pairs as complex numbers."""
    parts = [positions[:, a:a + 1].double() * theta ** (-torch.arange(n, dtype=torch.float64, device=x.device) / max(n, 1))
             for a, n in enumerate(sections)]
    angle = torch.cat(parts, dim=1)[:, None, :] * sign
    x = x.detach().double()
    if layout == "interleaved":
        a, b = x[..., 0::2], x[..., 1::2]
    else:
        a, b = x.chunk(2, dim=-1)
    u, v = a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()
    size = a.abs() + b.abs()
    if layout == "interleaved":
        return torch.stack([u, v], dim=-1).flatten(-2), torch.stack([size, size], dim=-1).flatten(-2)
    return torch.cat([u, v], dim=-1), torch.cat([size, size], dim=-1)


def rotate_bound(want, size, dtype):
    """Error of the FP32 rotation (angle within 2^-24 turns, sines within 2 ULP, three roundings: below 2^-20 of the
    pair) and of the rounding to ``dtype``."""
    unit = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    return size * 2.0 ** -20 + want.abs() * unit + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def attend(q, k_pages, v_pages, table, kv_lens, new, *, causal=False, window=None, sinks=0, scale=None):
    """Output, log-sum-exp and elementwise error bounds of paged attention, one session and head at a time in 64 bits.
    ``new``: new tokens of each session. Bounds: P is rounded to the 16-bit type (relative unit u, and for fp16 2^-25
    absolute below its normal range), the output once more; scores and sums are FP32, products accumulated with an error
    of at most 2^-22 of the sum of magnitudes each step."""
    page, kv_heads, d = k_pages.shape[1:]
    heads = q.shape[1]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    half = q.dtype == torch.float16
    unit = 2.0 ** -11 if half else 2.0 ** -8
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    out_bound, lse_bound = torch.zeros_like(out), torch.zeros_like(lse)
    first = 0
    for s, n in enumerate(new):
        total = int(kv_lens[s])
        held = table[s][:-(-total // page)].long() if total else table[s][:0].long()
        k = k_pages[held].flatten(0, 1)[:total].double()
        v = v_pages[held].flatten(0, 1)[:total].double()
        keys = torch.arange(total, device=q.device)
        last = torch.arange(total - n, total, device=q.device) if causal else torch.full((n,), total - 1, device=q.device)
        seen = keys <= last[:, None]
        if window is not None:
            seen &= (keys > last[:, None] - window) | (keys < sinks)
        some = seen.any(dim=1)
        for h in range(heads):
            x = q[first:first + n, h].double()
            kh, vh = k[:, h // (heads // kv_heads)], v[:, h // (heads // kv_heads)]
            unseen = ~seen.any(dim=0)  # what no token sees may hold anything
            kh, vh = kh.masked_fill(unseen[:, None], 0.0), vh.masked_fill(unseen[:, None], 0.0)
            if not total:
                continue
            score = (x @ kh.T * scale).masked_fill(~seen, -math.inf)
            top = score.amax(dim=1, keepdim=True).nan_to_num(neginf=0.0)
            p = torch.exp(score - top)
            total_p = p.sum(dim=1, keepdim=True).clamp(min=1e-300)
            rows = slice(first, first + n)
            out[rows, h] = p @ vh / total_p
            lse[rows, h] = torch.where(some, (top + total_p.log())[:, 0], -math.inf)
            weight = p @ vh.abs() / total_p
            noise = (x.abs() @ kh.abs().T * scale).masked_fill(~seen, 0.0).amax(dim=1, keepdim=True) * (d / 16 + 8) * 2.0 ** -22
            noise = noise + 2.0 ** -20 + total * 2.0 ** -24
            out_bound[rows, h] = unit * (weight + out[rows, h].abs()) * 1.01 + 2.0 * noise * weight
            if half:
                out_bound[rows, h] += 2.0 ** -24 + seen.sum(dim=1, keepdim=True) * 2.0 ** -25 * vh.abs().amax()
            lse_bound[rows, h] = noise[:, 0] + lse[rows, h].nan_to_num(neginf=0.0).abs() * 2.0 ** -22
        first += n
    return out, lse, out_bound, lse_bound


def within(got, want, bound):
    """Whether ``got`` is within ``bound`` of ``want`` everywhere (equal infinities count as equal)."""
    got = got.double()
    return bool(((got - want).abs() <= bound).logical_or(got == want).all())


def paged_batch(g, new, totals, kv_heads, d, page, dtype, *, device="cuda", extra=3, width_extra=0, fill=None, layout="nhd"):
    """Random pages of sessions of ``totals`` tokens, the last ``new`` of them new; pages in a random order. ``fill``:
    what positions that no session holds are filled with. ``layout="hnd"``: heads outside of tokens in memory."""
    counts = [-(-t // page) for t in totals]
    pages, width = sum(counts) + extra, max(max(counts), 1) + width_extra
    shape = (pages, page, kv_heads, d) if layout == "nhd" else (pages, kv_heads, page, d)
    made = []
    for _ in range(2):
        t = torch.randn(shape, generator=g, device=device).to(dtype)
        made.append(t if layout == "nhd" else t.transpose(1, 2))
    order = torch.randperm(pages, generator=g, device=device).to(torch.int32)
    table = torch.full((len(totals), width), -1, dtype=torch.int32, device=device)
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = order[at:at + n]
        at += n
    if fill is not None:
        held = torch.zeros(pages, page, dtype=torch.bool, device=device)
        for s, t in enumerate(totals):
            for b in range(counts[s]):
                held[int(table[s, b]), :min(page, t - b * page)] = True
        for t in made:
            t[~held] = fill
    return (*made, table, torch.tensor(totals, dtype=torch.int32, device=device),
            torch.tensor([0] + list(new), device=device).cumsum(0).to(torch.int32))


class ListTable:
    """The page table's rules in Python lists (and the moves that its data makes, on a CPU copy of the storage)."""

    def __init__(self, pages, seqs, width, page, storage):
        self.refs, self.lens = [0] * pages, [0] * seqs
        self.rows = [[-1] * width for _ in range(seqs)]
        self.page, self.storage = page, storage

    def _blocks(self, n):
        return -(-n // self.page)

    def _free(self):
        return [i for i, r in enumerate(self.refs) if r == 0]

    def allocate(self, seqs, lens):
        free = self._free()
        need = sum(self._blocks(n) - self._blocks(self.lens[s]) for s, n in zip(seqs, lens))
        bad = len(set(seqs)) < len(seqs) or any(n < self.lens[s] or self._blocks(n) > len(self.rows[s]) for s, n in zip(seqs, lens))
        if bad or need > len(free):
            return False
        for s, n in zip(seqs, lens):
            for b in range(self._blocks(self.lens[s]), self._blocks(n)):
                self.rows[s][b] = free.pop(0)
                self.refs[self.rows[s][b]] = 1
            self.lens[s] = n
        return True

    def fork(self, parents, children, lens):
        free = self._free()
        if len(set(children)) < len(children) or sum(n % self.page > 0 for n in lens) > len(free):
            return False
        if any(self.lens[c] or n > self.lens[p] for p, c, n in zip(parents, children, lens)):
            return False
        for p, c, n in zip(parents, children, lens):
            for b in range(n // self.page):
                self.rows[c][b] = self.rows[p][b]
                self.refs[self.rows[p][b]] += 1
            if n % self.page:
                b = n // self.page
                self.rows[c][b] = free.pop(0)
                self.refs[self.rows[c][b]] = 1
                self.storage[:, self.rows[c][b], :n % self.page] = self.storage[:, self.rows[p][b], :n % self.page]
            self.lens[c] = n
        return True

    def release(self, seqs):
        for s in seqs:
            for b, p in enumerate(self.rows[s]):
                if p >= 0:
                    self.refs[p] -= 1
                self.rows[s][b] = -1
            self.lens[s] = 0

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [i for i in range(live) if self.refs[i] == 0]
        movers = [i for i in range(live, len(self.refs)) if self.refs[i]]
        to = dict(zip(movers, holes))
        for src, dst in to.items():
            self.storage[:, dst] = self.storage[:, src]
            self.refs[dst], self.refs[src] = self.refs[src], 0
        self.rows = [[to.get(p, p) for p in row] for row in self.rows]
        return live

    def check(self, table, storage):
        assert table.refcount.tolist() == self.refs
        assert table.lens.tolist() == self.lens
        assert table.block_table.tolist() == self.rows
        assert torch.equal(storage.cpu(), self.storage)
