"""The paged KV cache as a user has it: sessions that fork, rewind and end, and the video DiT over it."""

import importlib.util
from pathlib import Path

import pytest
import torch

from .paged_support import attend, spun

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _checked(cuda_device):
    from reelcache_b200.ops import _ext
    yield
    _ext.check_status(cuda_device)


def _cache(**kw):
    from reelcache_b200.paged_cache import PagedKVCache
    return PagedKVCache(2, 2, 64, **{"pages": 24, "page_size": 16, "max_sessions": 6, "max_tokens": 128, **kw})


def test_sessions_follow_their_own_histories():
    """Forks, rewinds, ends and compactions against histories kept as plain tensors."""
    from reelcache_b200.ops.rope import AxisRope
    g = torch.Generator(device="cuda").manual_seed(0)
    rope = AxisRope.wan(64)
    cache = _cache()
    plain = {}  # slot -> per layer (k, v) [tokens, 2, 64]
    empty = lambda: [(torch.zeros(0, 2, 64, device="cuda").bfloat16(),) * 2 for _ in range(2)]  # noqa: E731

    def step(pairs, causal):
        batch = cache.extend(pairs)
        rows = batch.tokens
        positions = torch.randint(0, 900, (rows, 3), generator=g, device="cuda", dtype=torch.int32)
        for layer in range(2):
            q, k, v = (torch.randn(rows, h, 64, generator=g, device="cuda").bfloat16() for h in (4, 2, 2))
            turned = cache.append(layer, batch, q, k, v, positions, rope)
            out = cache.attend(layer, batch, turned, causal=causal)
            at = 0
            for s, n in pairs:
                want_k = spun(k[at:at + n], positions[at:at + n], rope.sections, 10000.0, "interleaved")[0]
                have = plain[s.slot][layer]
                plain[s.slot][layer] = (torch.cat([have[0], want_k.bfloat16()]), torch.cat([have[1], v[at:at + n]]))
                kv = plain[s.slot][layer]
                table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
                want = attend(turned[at:at + n], kv[0][None], kv[1][None], table, [kv[0].shape[0]], [n], causal=causal)[0]
                assert float((out[at:at + n].double() - want).norm() / want.norm().clamp(min=1e-9)) < 1e-2
                at += n

    a = cache.open()
    plain[a.slot] = empty()
    step([(a, 37)], False)
    b, c = cache.fork(a, [37, 20])
    for s, n in ((b, 37), (c, 20)):
        plain[s.slot] = [(k[:n], v[:n]) for k, v in plain[a.slot]]
    assert cache.pages - cache.free_pages == 3 + 1 + 1  # three pages, and a copied tail for each fork
    step([(a, 1), (b, 1), (c, 1)], True)
    step([(c, 30), (a, 16)], True)
    cache.close(a)
    assert cache.compact() == cache.pages - cache.free_pages
    step([(b, 40), (c, 5)], False)
    (d,) = cache.fork(b)
    plain[d.slot] = [tuple(kv) for kv in plain[b.slot]]
    step([(d, 3), (b, 11), (c, 2)], True)
    cache.close(b, c, d)
    assert cache.free_pages == cache.pages and int(cache.table.refcount.abs().sum()) == 0


def test_refusals():
    from reelcache_b200.errors import CapacityError, ConfigurationError, StateError, UnsupportedError
    from reelcache_b200.paged_cache import PagedKVCache
    for wrong in (dict(page_size=12), dict(pages=0), dict(max_sessions=0), dict(max_tokens=0)):
        with pytest.raises(ConfigurationError):
            _cache(**wrong)
    with pytest.raises(UnsupportedError):
        _cache(device="cpu")
    with pytest.raises(ConfigurationError):
        PagedKVCache(1, 1, 96, pages=1, page_size=8, max_sessions=1, max_tokens=8)
    cache = _cache(pages=6, max_sessions=3)
    a, b = cache.open(), cache.open()
    cache.extend([(a, 40), (b, 16)])
    with pytest.raises(CapacityError):
        cache.extend([(a, 30), (b, 30)])
    with pytest.raises(CapacityError):
        cache.extend([(a, 100)])
    with pytest.raises(StateError):
        cache.extend([(a, 1), (a, 1)])
    with pytest.raises(ConfigurationError):
        cache.fork(a, [41])
    with pytest.raises(CapacityError):
        cache.fork(a, [40, 40])  # one slot left
    (c,) = cache.fork(a, [32])
    with pytest.raises(StateError):
        cache.again([(c, 8)])  # those rows are a's too
    with pytest.raises(CapacityError):
        cache.open()
    cache.close(a)
    for call in (lambda: cache.close(a), lambda: cache.extend([(a, 1)]), lambda: cache.fork(a), lambda: cache.close(b, b)):
        with pytest.raises(StateError):
            call()
    cache.again([(c, 8)])  # now its own
    assert cache.free_pages == 3


def test_dit_over_pages_equals_the_dense_cache():
    """The newest chunk of forked sessions in one batched forward, against the contiguous cache session by session."""
    from reelcache_b200.models.causal_wan import CAUSVID, CausalWanDiT, KVCache
    from reelcache_b200.paged_cache import PagedKVCache
    cfg = CAUSVID.scaled(layers=2, dim=256, heads=2, ffn=512, text_dim=128, text_len=16, latent_height=8, latent_width=16)
    model = CausalWanDiT(cfg, "cuda", seed=3)
    text_kv = model.encode_text(torch.randn(cfg.text_len, cfg.text_dim, device="cuda"))
    torch.manual_seed(0)
    draw = lambda: torch.randn(cfg.in_dim, cfg.frames_per_chunk, cfg.latent_height, cfg.latent_width, device="cuda")  # noqa: E731
    first, second, left, right = (draw() for _ in range(4))
    cache = PagedKVCache(cfg.layers, cfg.heads, cfg.head_dim, pages=40, page_size=cfg.tokens_per_frame, max_sessions=4,
                         max_tokens=4 * cfg.chunk_tokens)
    root = cache.open()
    captured = {}
    for x in (first, second):
        batch = cache.extend([(root, cfg.chunk_tokens)])
        model.forward_sessions(x[None], 500.0, cache, batch, text_kv, capture=lambda l, k, v: captured.__setitem__(l, (k.clone(), v.clone())))
    a, b = cache.fork(root, [2 * cfg.chunk_tokens, cfg.chunk_tokens])
    batch = cache.extend([(a, cfg.chunk_tokens), (b, cfg.chunk_tokens)])
    got = model.forward_sessions(torch.stack([left, right]), 250.0, cache, batch, text_kv)
    for latents, history, out in ((left, [first, second], got[0]), (right, [first], got[1])):
        dense = KVCache(cfg, 4, "cuda")
        kept = {}
        for i, x in enumerate(history):
            model.forward_chunk(x, 500.0, i, dense, text_kv, capture=lambda l, k, v: kept.__setitem__(l, (k.clone(), v.clone())))
        if len(history) == 2:
            for layer in range(cfg.layers):
                for x, y in zip(captured[layer], kept[layer]):
                    assert float((x.float() - y.float()).norm() / y.float().norm()) < 1e-2
        want = model.forward_chunk(latents, 250.0, len(history), dense, text_kv)
        assert float((out - want).norm() / want.norm()) < 2e-2
    with pytest.raises(ValueError):
        model.forward_sessions(left[None], 250.0, cache, cache.extend([(root, 5)]), text_kv)


def test_example_runs():
    path = Path(__file__).resolve().parents[1] / "examples" / "paged_sessions.py"
    spec = importlib.util.spec_from_file_location("paged_sessions", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    from reelcache_b200.models.causal_wan import CAUSVID
    report = module.run(CAUSVID.scaled(**module.SMALL), chunks=3, branches=4, steps=1)
    assert report["history_pages"] == 9 and report["pages_after_forks"] == 9 and report["pages_if_copied"] == 30
    assert report["batched_vs_separate_difference"] < 2e-2
    assert report["pages_after_compaction"] == 9 + 2 * 3 and report["pages_used_at_the_end"] == 9 + 4 * 3


# -- batches that are out of date -------------------------------------------------------------------------------------

def _rows(n, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v = (torch.randn(n, h, 64, generator=g, device="cuda").bfloat16() for h in (4, 2, 2))
    return q, k, v, torch.zeros(n, 3, dtype=torch.int32, device="cuda")


def test_a_batch_of_a_closed_session_is_refused():
    """Its pages may be another session's by now."""
    from reelcache_b200.errors import StateError
    from reelcache_b200.ops.rope import AxisRope
    rope = AxisRope.wan(64)
    cache = _cache()
    a = cache.open()
    old = cache.extend([(a, 20)])
    cache.append(0, old, *_rows(20), rope)
    cache.close(a)
    b = cache.open()
    batch = cache.extend([(b, 20)])
    cache.append(0, batch, *_rows(20, 1), rope)
    before = cache.storage.clone()
    q = _rows(20)[0]
    for call in (lambda: cache.append(0, old, *_rows(20, 2), rope), lambda: cache.attend(0, old, q)):
        with pytest.raises(StateError):
            call()
    assert torch.equal(cache.storage, before)
    cache.attend(0, batch, q)


def test_a_batch_from_before_a_compaction_is_refused():
    from reelcache_b200.errors import StateError
    from reelcache_b200.ops.rope import AxisRope
    rope = AxisRope.wan(64)
    cache = _cache()
    a, b = cache.open(), cache.open()
    cache.extend([(a, 40)])
    batch = cache.extend([(b, 20)])
    cache.append(0, batch, *_rows(20), rope)
    cache.close(a)
    cache.compact()
    before = cache.storage.clone()
    for call in (lambda: cache.append(0, batch, *_rows(20, 2), rope), lambda: cache.attend(0, batch, _rows(20)[0])):
        with pytest.raises(StateError):
            call()
    assert torch.equal(cache.storage, before)
    batch = cache.again([(b, 20)])
    cache.append(0, batch, *_rows(20, 2), rope)
    cache.attend(0, batch, _rows(20)[0])


@pytest.mark.parametrize("lengths,refused", [([48], True), ([45], True), ([33], True), ([32], False), ([31], False), ([17], False),
                                             ([48, 17], True), ([17, 48], True), ([], False)])
def test_a_batch_whose_tokens_were_forked_is_refused(lengths, refused):
    """After a fork that took some of the batch's new tokens (16 of 48 here: a page of their own, or the copied rows of a
    page), writing them would change the child's history or leave its copy behind."""
    from reelcache_b200.errors import StateError
    from reelcache_b200.ops.rope import AxisRope
    rope = AxisRope.wan(64)
    cache = _cache()
    a = cache.open()
    cache.append(0, cache.extend([(a, 32)]), *_rows(32), rope)
    batch = cache.extend([(a, 16)])
    children = cache.fork(a, lengths)
    if not refused:
        cache.append(0, batch, *_rows(16), rope)
    else:
        before = cache.storage.clone()
        with pytest.raises(StateError):
            cache.append(0, batch, *_rows(16), rope)
        assert torch.equal(cache.storage, before)
    cache.attend(0, batch, _rows(16)[0])  # reading is not writing
    cache.close(*children)
    cache.append(0, cache.again([(a, 16)]), *_rows(16), rope)


def test_a_batch_inside_a_page_that_was_forked_before_it():
    """Rows before the batch's tokens in the same page may have been copied, at any time."""
    from reelcache_b200.errors import StateError
    from reelcache_b200.ops.rope import AxisRope
    rope = AxisRope.wan(64)
    cache = _cache()
    a = cache.open()
    cache.append(0, cache.extend([(a, 20)]), *_rows(20), rope)
    cache.fork(a, [20])
    batch = cache.extend([(a, 6)])  # tokens 20 to 25
    cache.append(0, batch, *_rows(6), rope)
    cache.fork(a, [18])
    cache.append(1, batch, *_rows(6), rope)
    (c,) = cache.fork(a, [21])
    with pytest.raises(StateError):
        cache.append(0, batch, *_rows(6), rope)
    cache.append(0, cache.again([(a, 6)]), *_rows(6), rope)  # once more, by intent
    cache.append(0, cache.extend([(a, 3)]), *_rows(3), rope)
    cache.append(0, cache.extend([(c, 3)]), *_rows(3), rope)


def test_a_batch_of_another_cache_is_refused():
    from reelcache_b200.errors import StateError
    from reelcache_b200.ops.rope import AxisRope
    rope = AxisRope.wan(64)
    cache, other = _cache(), _cache()
    batch = cache.extend([(cache.open(), 20)])
    for call in (lambda: other.append(0, batch, *_rows(20), rope), lambda: other.attend(0, batch, _rows(20)[0])):
        with pytest.raises(StateError):
            call()


def test_a_later_extension_leaves_a_batch_as_it_is():
    """A batch from before its session's next extension names the same tokens, and the model rotates them at their place."""
    from reelcache_b200.models.causal_wan import CAUSVID, CausalWanDiT
    from reelcache_b200.paged_cache import PagedKVCache
    cfg = CAUSVID.scaled(layers=2, dim=256, heads=2, ffn=512, text_dim=128, text_len=16, latent_height=8, latent_width=16)
    model = CausalWanDiT(cfg, "cuda", seed=3)
    text_kv = model.encode_text(torch.randn(cfg.text_len, cfg.text_dim, device="cuda"))
    cache = PagedKVCache(cfg.layers, cfg.heads, cfg.head_dim, pages=40, page_size=cfg.tokens_per_frame, max_sessions=4,
                         max_tokens=4 * cfg.chunk_tokens)
    a = cache.open()
    x = torch.randn(1, cfg.in_dim, cfg.frames_per_chunk, cfg.latent_height, cfg.latent_width, device="cuda")
    model.forward_sessions(x, 500.0, cache, cache.extend([(a, cfg.chunk_tokens)]), text_kv)
    batch = cache.extend([(a, cfg.chunk_tokens)])
    want = model.forward_sessions(x, 500.0, cache, batch, text_kv)
    kept = cache.storage.clone()
    cache.extend([(a, cfg.chunk_tokens)])
    assert torch.equal(model.forward_sessions(x, 500.0, cache, batch, text_kv), want)
    assert torch.equal(cache.storage, kept)


def test_fewer_rows_than_new_tokens_are_refused():
    """The lengths count all new tokens, so a shorter call would put the ones it has in the wrong places."""
    from reelcache_b200.errors import ConfigurationError
    from reelcache_b200.ops.rope import AxisRope
    cache = _cache()
    batch = cache.extend([(cache.open(), 20), (cache.open(), 7)])
    before = cache.storage.clone()
    for call in (lambda: cache.append(0, batch, *_rows(26), AxisRope.wan(64)), lambda: cache.attend(0, batch, _rows(20)[0])):
        with pytest.raises(ConfigurationError):
            call()
    assert torch.equal(cache.storage, before)
    cache.append(0, batch, *_rows(30), AxisRope.wan(64))  # rows past the batch's belong to no session
    cache.attend(0, batch, _rows(30)[0])


def test_books_stay_as_they_were_when_a_call_fails(monkeypatch):
    """An exception on the way to the device leaves the host's counts, slots and lengths alone."""
    from reelcache_b200.ops import paged
    cache = _cache()
    a = cache.open()
    cache.extend([(a, 20)])
    books = lambda: (cache.free_pages, list(cache._free_slots), a.length, len(a.blocks), [b.holders for b in a.blocks], a.open)  # noqa: E731
    before, state = books(), cache.table.state.clone()

    def fails(*args, **kw):
        raise RuntimeError("no memory")

    for name, call in (("allocate", lambda: cache.extend([(a, 30)])), ("fork", lambda: cache.fork(a, [20, 3])),
                       ("release", lambda: cache.close(a))):
        for target, attribute in ((paged.PageTable, name), (type(cache), "_ints")):
            with monkeypatch.context() as patch:
                patch.setattr(target, attribute, fails)
                with pytest.raises(RuntimeError, match="no memory"):
                    call()
            assert books() == before and torch.equal(cache.table.state, state)
    cache.fork(a, [20, 3])
    cache.extend([(a, 30)])
    cache.close(a)


def test_sizes_that_the_page_table_cannot_hold_are_refused_at_once():
    from reelcache_b200.errors import ConfigurationError
    for wrong in (dict(page_size=65536 + 8, max_tokens=65536 + 8, pages=1), dict(pages=1 << 20, page_size=8), dict(max_sessions=1 << 20, max_tokens=8)):
        with pytest.raises(ConfigurationError):
            _cache(**wrong)


def test_dit_over_pages_writes_the_dense_caches_rows():
    """Keys and values of the first layer, whose input is the same on both paths, are the dense cache's bit for bit: one
    rounding after norm and rotation."""
    from reelcache_b200.models.causal_wan import CAUSVID, CausalWanDiT, KVCache
    from reelcache_b200.paged_cache import PagedKVCache
    cfg = CAUSVID.scaled(layers=1, dim=256, heads=2, ffn=512, text_dim=128, text_len=16, latent_height=8, latent_width=16)
    model = CausalWanDiT(cfg, "cuda", seed=5)
    text_kv = model.encode_text(torch.randn(cfg.text_len, cfg.text_dim, device="cuda"))
    chunk = cfg.chunk_tokens
    cache = PagedKVCache(1, cfg.heads, cfg.head_dim, pages=60, page_size=16, max_sessions=3, max_tokens=4 * chunk)
    sessions = [cache.open() for _ in range(2)]
    cache.extend([(sessions[1], 2 * chunk)])  # the second session is at its third chunk
    batch = cache.extend([(s, chunk) for s in sessions])
    x = torch.randn(2, cfg.in_dim, cfg.frames_per_chunk, cfg.latent_height, cfg.latent_width, device="cuda")
    captured = {}
    model.forward_sessions(x, 500.0, cache, batch, text_kv, capture=lambda l, k, v: captured.__setitem__(l, (k.clone(), v.clone())))
    for i, (s, index) in enumerate(zip(sessions, (0, 2))):
        dense, kept = KVCache(cfg, 3, "cuda"), {}
        model.forward_chunk(x[i], 500.0, index, dense, text_kv, capture=lambda l, k, v: kept.__setitem__(l, (k.clone(), v.clone())))
        at = torch.arange(index * chunk, (index + 1) * chunk, device="cuda")
        pages = batch.table[i, at // 16].long()
        for which, rows in enumerate((dense.rows(0, "K"), dense.rows(0, "V"))):
            assert torch.equal(cache.storage[0, which, pages, at % 16].flatten(1), rows[at])
            assert torch.equal(captured[0][which][i * chunk:(i + 1) * chunk], kept[0][which])


def test_new_rows_are_where_append_writes():
    """The rows that a kernel of its own writes are those of append; the model's rotation from positions is its tables'."""
    from reelcache_b200.models.causal_wan import CAUSVID, CausalWanDiT
    from reelcache_b200.paged_cache import PagedKVCache
    cfg = CAUSVID.scaled(layers=1, dim=256, heads=2, ffn=512, text_dim=128, text_len=16, latent_height=8, latent_width=16)
    model = CausalWanDiT(cfg, "cuda", seed=5)
    cache = PagedKVCache(1, cfg.heads, cfg.head_dim, pages=60, page_size=24, max_sessions=4, max_tokens=4 * cfg.chunk_tokens)
    a, b, c = (cache.open() for _ in range(3))
    cache.extend([(b, cfg.chunk_tokens)])
    batch = cache.extend([(a, cfg.chunk_tokens), (c, 0), (b, cfg.chunk_tokens)])
    positions = model.session_positions([0, 1])
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(batch.tokens, cfg.heads, cfg.head_dim, generator=g, device="cuda").bfloat16() for _ in range(3))
    cache.append(0, batch, q, k, v, positions, model.axis_rope)
    rows = cache.new_rows(batch)
    assert torch.equal(cache.token_rows(0, "V")[rows], v.flatten(1))
    cos, sin = (t[:, None].double() for t in model.session_rope([0, 1]))
    x, y = k.double()[..., 0::2], k.double()[..., 1::2]
    want = torch.stack([x * cos - y * sin, x * sin + y * cos], dim=-1).flatten(1)
    size = torch.stack([x.abs() + y.abs()] * 2, dim=-1).flatten(1)  # tables in FP32, the rotation's sines within 2^-20, bf16
    assert bool(((cache.token_rows(0, "K")[rows].double() - want).abs() <= size * 2.0 ** -19 + want.abs() * 2.0 ** -8).all())
    for i, index in enumerate((0, 1)):
        for got, table in zip(model.session_rope([0, 1]), model.token_rope(index)):
            assert torch.equal(got[i * cfg.chunk_tokens:(i + 1) * cfg.chunk_tokens], table)
    far = model.session_rope([model.rope.rows])  # beyond the model's own table
    assert far[0].shape == (cfg.chunk_tokens, cfg.head_dim // 2) and bool((far[0] ** 2 + far[1] ** 2 - 1).abs().max() < 1e-6)
    cache.fork(b)
    with pytest.raises(Exception, match="forked"):
        cache.new_rows(batch)


def test_a_session_of_another_cache_is_refused():
    """Its slot and pages are other ones here."""
    from reelcache_b200.errors import StateError
    cache, other = _cache(), _cache()
    a, b = cache.open(), other.open()
    other.extend([(b, 20)])
    (c,) = other.fork(b)
    state = cache.table.state.clone()
    for call in (lambda: cache.extend([(a, 3), (b, 3)]), lambda: cache.extend([(c, 3)]), lambda: cache.fork(b), lambda: cache.close(b),
                 lambda: cache.again([(b, 3)])):
        with pytest.raises(StateError):
            call()
    assert torch.equal(cache.table.state, state) and a.length == 0 and cache.free_pages == cache.pages
    other.close(b, c)


def test_rows_are_the_pages_token_rows():
    """A restored chunk can be written straight into a session's pages."""
    cache = _cache()
    a = cache.open()
    batch = cache.extend([(a, 40)])
    k, v = (torch.randn(40, 2, 64, device="cuda").bfloat16() for _ in range(2))
    for block in range(3):
        page, n = int(batch.table[0, block]), min(16, 40 - 16 * block)
        for which, rows in (("K", k), ("V", v)):
            cache.rows(1, which, page)[:n] = rows[16 * block:16 * block + n].flatten(1)
    q = torch.randn(40, 4, 64, device="cuda").bfloat16()
    out = cache.attend(1, batch, q)
    want = attend(q, k[None], v[None], torch.zeros(1, 1, dtype=torch.int32, device="cuda"), [40], [40])[0]
    assert float((out.double() - want).norm() / want.norm()) < 1e-2


def test_example_decodes_token_by_token():
    """Forked sessions that append and attend a token at a time against one pass over each whole sequence; the tails of 100
    prompt tokens (7 pages of 16) are copied, 12 tokens take a page more at most."""
    path = Path(__file__).resolve().parents[1] / "examples" / "paged_sessions.py"
    spec = importlib.util.spec_from_file_location("paged_sessions", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    for heads, kv_heads, branches in ((8, 2, 3), (4, 4, 1)):
        difference, beyond = module.decode(heads=heads, kv_heads=kv_heads, branches=branches)
        assert difference < 2e-2 and beyond == branches
