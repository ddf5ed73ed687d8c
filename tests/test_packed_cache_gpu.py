"""The paged cache in 8 bits, and attention over chosen blocks of it, as a user has them: sessions that fork, rewind and end, and
the video DiT over them."""

import importlib.util
from pathlib import Path

import pytest
import torch

from .paged_support import attend, spun, within
from .sparse_support import held, quantise

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _checked(cuda_device):
    from reelcache_b200.ops import _ext
    yield
    _ext.check_status(cuda_device)


def _cache(**kw):
    from reelcache_b200.paged_cache import PagedKVCache
    return PagedKVCache(2, 2, 64, **{"pages": 40, "page_size": 24, "max_sessions": 6, "max_tokens": 200, **kw})


def _values(rows):
    codes, power = quantise(rows, BF16)
    return (codes * torch.exp2(power.double())[..., None]).to(BF16)


def _blocks_of(rows, q, n, block, keep, query_block, recent, causal):
    """Keys that each query block and KV head sees, by the definition, from a session's own rows."""
    total = rows.shape[0]
    for start in range(0, n, query_block):
        count = min(query_block, n - start)
        end = total - n + start + count if causal else total
        high = max(0, total - n + (start if causal else 0) - recent) // block
        for h in range(rows.shape[1]):
            means = torch.stack([rows[b * block:(b + 1) * block, h].double().mean(dim=0) for b in range(high)]).to(BF16).double() if high else None
            best = []
            if high:
                pooled = q[start:start + count, 2 * h:2 * h + 2].double().sum(dim=0)
                best = torch.sort((means @ pooled.T).amax(dim=1), descending=True, stable=True).indices[:keep].sort().values.tolist()
            yield start, count, h, [p for b in best for p in range(b * block, (b + 1) * block)] + list(range(high * block, end))


@pytest.mark.parametrize("packed", [False, True])
def test_sessions_follow_their_own_histories(packed):
    """Forks inside a page and a block, rewinds, ends and compactions against histories kept as plain tensors: dense attention, and
    attention over chosen blocks, whose means follow the pages."""
    from reelcache_b200.ops.rope import AxisRope
    g = torch.Generator(device="cuda").manual_seed(0)
    rope = AxisRope.wan(64)
    cache = _cache(packed=packed, block=8)
    plain = {}  # slot -> per layer (k, v) [tokens, 2, 64]
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")

    def step(pairs, causal, query_block=1):
        batch = cache.extend(pairs)
        for layer in range(2):
            positions = torch.randint(0, 900, (batch.tokens, 3), generator=g, device="cuda", dtype=torch.int32)
            q, k, v = (torch.randn(batch.tokens, h, 64, generator=g, device="cuda").bfloat16() for h in (4, 2, 2))
            if packed and layer == 1:  # rows as they are
                turned = q
                cache.store(layer, batch, k, v)
            else:
                turned = cache.append(layer, batch, q, k, v, positions, rope)
            dense = cache.attend(layer, batch, turned, causal=causal)
            chosen = cache.attend(layer, batch, turned, causal=causal, keep=3, query_block=query_block, recent=9)
            k_pages, v_pages = cache.layer_pages(layer)
            new = [x.flatten(0, 1)[_rows(cache, batch)] for x in ((held(k_pages, BF16), held(v_pages, BF16)) if packed else (k_pages, v_pages))]
            if layer == 0:
                want = spun(k, positions, rope.sections, 10000.0, "interleaved")[0]
                assert bool(((new[0].double() - want).abs() <= want.abs() * 2.0 ** (-4 if packed else -8) + 2.0 ** -8).all())
            assert torch.equal(new[1], _values(v) if packed else v)
            at = 0
            for s, n in pairs:
                have = plain[s.slot][layer]
                kv = plain[s.slot][layer] = tuple(torch.cat([x, y[at:at + n]]) for x, y in zip(have, new))
                total = kv[0].shape[0]
                want, _, bound, _ = attend(turned[at:at + n], kv[0][None], kv[1][None], table, [total], [n], causal=causal)
                extra = total * 2.0 ** -24 * float(kv[1].abs().max())
                assert within(dense[at:at + n], want, bound + extra)
                for start, count, h, keys in _blocks_of(kv[0], turned[at:at + n], n, 8, 3, query_block, 9, causal):
                    rows = slice(at + start, at + start + count)
                    want, _, bound, _ = attend(turned[rows, 2 * h:2 * h + 2], *(x[keys, h][None, :, None] for x in kv), table, [len(keys)], [count], causal=causal)
                    assert within(chosen[rows, 2 * h:2 * h + 2], want, bound + extra)
                at += n

    a = cache.open()
    plain[a.slot] = [(torch.zeros(0, 2, 64, device="cuda").bfloat16(),) * 2 for _ in range(2)]
    step([(a, 61)], False, 16)
    b, c = cache.fork(a, [61, 30])  # inside a page and a block, 30 in the middle of one
    for s, n in ((b, 61), (c, 30)):
        plain[s.slot] = [tuple(x[:n] for x in kv) for kv in plain[a.slot]]
    step([(a, 1), (b, 1), (c, 1)], True)
    step([(c, 30), (a, 16)], True, 5)
    cache.close(a)
    assert cache.compact() == cache.pages - cache.free_pages
    step([(b, 40), (c, 5)], False, 64)
    (d,) = cache.fork(b)
    plain[d.slot] = [tuple(kv) for kv in plain[b.slot]]
    step([(d, 3), (b, 11), (c, 2)], True, 2)
    if packed:
        for layer in range(2):
            k, v = cache.read(layer, [c, d])
            want = [torch.cat([plain[s.slot][layer][i] for s in (c, d)]) for i in range(2)]
            assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    cache.close(b, c, d)
    assert cache.free_pages == cache.pages


def _rows(cache, batch):
    """Places of the batch's new tokens in the layer's rows."""
    out = []
    for s, n, length in zip(range(len(batch.counts)), batch.counts, batch.lengths):
        out += [int(batch.table[s, at // cache.page_size]) * cache.page_size + at % cache.page_size for at in range(length - n, length)]
    return torch.tensor(out, device="cuda")


def test_a_rewritten_chunk_has_new_means():
    """A further denoising step writes the chunk again: its blocks' means are those of the new rows."""
    from reelcache_b200.ops.rope import AxisRope
    g = torch.Generator(device="cuda").manual_seed(1)
    cache = _cache(block=24, packed=True)
    a = cache.open()
    rope = AxisRope.wan(64)
    rows = lambda n: (*(torch.randn(n, h, 64, generator=g, device="cuda").bfloat16() for h in (4, 2, 2)),  # noqa: E731
                      torch.zeros(n, 3, dtype=torch.int32, device="cuda"))
    cache.append(0, cache.extend([(a, 30)]), *rows(30), rope)
    batch = cache.extend([(a, 50)])
    for _ in range(2):
        cache.append(0, batch, *rows(50), rope)
    k, _ = cache.read(0, [a])
    pages = cache.table.block_table[a.slot, :4].long()
    want = torch.stack([k[b * 24:min(80, (b + 1) * 24)].double().mean(dim=0) for b in range(4)]).to(BF16)
    assert torch.equal(cache.means[0, pages, 0], want)


def test_refusals():
    from reelcache_b200.errors import ConfigurationError, StateError, UnsupportedError
    for wrong in (dict(block=16), dict(block=4), dict(block=0), dict(block=48)):
        with pytest.raises(ConfigurationError):
            _cache(**wrong)
    plain, packed = _cache(), _cache(packed=True, block=8)
    rows = torch.randn(20, 2, 64, device="cuda").to(BF16)
    q = torch.randn(20, 4, 64, device="cuda").to(BF16)
    a, b = plain.open(), packed.open()
    one, two = plain.extend([(a, 20)]), packed.extend([(b, 20)])
    for call in (lambda: plain.store(0, one, rows, rows), lambda: plain.read(0, [a]), lambda: plain.attend(0, one, q, keep=2),
                 lambda: packed.token_rows(0, "K"), lambda: packed.rows(0, "V", 0)):
        with pytest.raises(UnsupportedError):
            call()
    for call in (lambda: packed.attend(0, two, q, keep=2, window=8), lambda: packed.attend(0, two, q, recent=8), lambda: packed.attend(0, two, q, query_block=4),
                 lambda: packed.store(0, two, rows.half(), rows.half()), lambda: packed.attend(0, two, q.half()), lambda: packed.store(0, two, rows[:3], rows[:3])):
        with pytest.raises(ConfigurationError):
            call()
    for call in (lambda: packed.read(0, []), lambda: packed.read(0, [a]), lambda: packed.store(0, one, rows, rows)):
        with pytest.raises(StateError):
            call()
    children = packed.fork(b, [20])
    with pytest.raises(StateError):
        packed.store(0, two, rows, rows)  # the fork has its rows
    packed.close(*children)


def _model(layers=2):
    from reelcache_b200.models.causal_wan import CAUSVID, CausalWanDiT
    return CausalWanDiT(CAUSVID.scaled(layers=layers, dim=256, heads=2, ffn=512, text_dim=128, text_len=16, latent_height=8, latent_width=16), "cuda", seed=3)


def _forward(model, cache, **how):
    g = torch.Generator(device="cuda").manual_seed(4)
    cfg = model.cfg
    draw = lambda n: torch.randn(n, cfg.in_dim, cfg.frames_per_chunk, cfg.latent_height, cfg.latent_width, device="cuda", generator=g)  # noqa: E731
    text = model.encode_text(torch.randn(cfg.text_len, cfg.text_dim, device="cuda", generator=g))
    root = cache.open()
    for _ in range(2):
        model.forward_sessions(draw(1), 0.0, cache, cache.extend([(root, cfg.chunk_tokens)]), text, **how)
    forks = cache.fork(root, count=2)
    return model.forward_sessions(draw(2), 500.0, cache, cache.extend([(s, cfg.chunk_tokens) for s in forks]), text, **how)


def test_model_over_a_packed_cache_sees_what_it_holds():
    """The forward over packed pages against the forward over 16-bit pages whose rows are rounded to the same numbers."""
    from reelcache_b200.paged_cache import PagedKVCache

    class Rounded(PagedKVCache):
        def rows_written(self, layer, batch):
            at = _rows(self, batch)
            for which in ("K", "V"):
                rows = self.token_rows(layer, which)
                rows[at] = _values(rows[at].unflatten(1, (2, 128))).flatten(1)

    model = _model()
    sizes = dict(pages=8 * model.cfg.frames_per_chunk, page_size=model.cfg.tokens_per_frame, max_sessions=3, max_tokens=4 * model.cfg.chunk_tokens)
    plain = _forward(model, Rounded(2, 2, 128, **sizes))
    packed = _forward(model, PagedKVCache(2, 2, 128, packed=True, **sizes))
    assert torch.equal(packed, plain)


@pytest.mark.parametrize("packed", [False, True])
def test_model_over_chosen_blocks(packed):
    """All of the past chosen gives the dense forward but for the order of sums; some of it, another one, every time the same."""
    from reelcache_b200.paged_cache import PagedKVCache
    model = _model(layers=1)
    sizes = dict(pages=8 * model.cfg.frames_per_chunk, page_size=model.cfg.tokens_per_frame, max_sessions=3, max_tokens=4 * model.cfg.chunk_tokens)
    make = lambda: PagedKVCache(1, 2, 128, packed=packed, block=8, **sizes)  # noqa: E731
    dense = _forward(model, make())
    whole = _forward(model, make(), sparse=dict(keep=1000, query_block=32))
    # attention's output is off by 2^-7 of its size at most either way (P and the output rounded to bf16), and the rest of a block, a
    # residual stream and a head, passes it on
    assert float((whole - dense).norm() / dense.norm()) < 2 * 2.0 ** -7
    some = _forward(model, make(), sparse=dict(keep=2, query_block=32))
    assert torch.equal(some, _forward(model, make(), sparse=dict(keep=2, query_block=32)))
    assert bool(some.isfinite().all()) and not torch.equal(some, whole)


@pytest.mark.parametrize("options", [["--packed"], ["--keep", "2"], ["--packed", "--keep", "2"]])
def test_example_runs(options, capsys):
    import json
    path = Path(__file__).resolve().parents[1] / "examples" / "paged_sessions.py"
    spec = importlib.util.spec_from_file_location("paged_sessions_example", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    example.main(["--small", "--chunks", "2", "--branches", "2", *options])
    got = json.loads(capsys.readouterr().out)
    assert got["packed"] == ("--packed" in options) and got["page_bytes"] > 0


def test_batches_without_new_tokens():
    cache = _cache(packed=True, block=8)
    a = cache.open()
    rows = torch.randn(30, 2, 64, device="cuda").to(BF16)
    cache.store(0, cache.extend([(a, 30)]), rows, rows)
    batch = cache.extend([(a, 0)])
    none = torch.zeros(0, 4, 64, dtype=BF16, device="cuda")
    cache.store(0, batch, none[:, :2], none[:, :2])
    assert cache.attend(0, batch, none).shape == none.shape
    assert cache.attend(0, batch, none, keep=2).shape == none.shape
    assert torch.equal(cache.read(0, [a])[0], _values(rows))
