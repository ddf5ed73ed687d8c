"""A paged KV cache's operators on sm_100a: writing new tokens (csrc/paged/rotate.cu, in 8 bits pack.cu), attending over the
pages (attend_short.cu, attend_chunk.cu, in 8 bits attend_packed.cu and expand.cu), choosing the blocks of sparse attention
(select.cu) and the page table (table.cu).

Pages: ``k_pages, v_pages [pages, page_size, kv_heads, head_dim]`` of one layer (any 16-byte aligned strides; the page
size is a multiple of 8 tokens). A batch of sequences is described by ``block_table [seqs, width]`` (page of each block
of ``page_size`` tokens, -1 for none), ``kv_lens [seqs]`` (tokens held, the new ones included) and ``cu_q [seqs + 1]``
(where each sequence's new tokens begin in ``q``), all int32 on the device (rows of the table may be strided: a slice
``table[:, :n]`` will do): nothing is read back, every call can be captured in a graph. Sequence ``s``'s new tokens are
its last ``cu_q[s + 1] - cu_q[s]`` positions.

Pages may hold their rows in 8 bits (:class:`PackedPages`): :func:`append`, :func:`attention` and :func:`block_means` take
either kind. Sparse attention is a choice of blocks for every few queries (:func:`select_blocks`) and attention over the
blocks as pages (:func:`blocks`), with a block table for each KV head.

Calls with page numbers outside the pool, lengths that do not fit their tensors or bounds, or page-table calls that cannot
be served, do nothing out of bounds and are reported by :func:`reelcache_b200.ops._ext.check_status`.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from ..errors import ConfigurationError, UnsupportedError
from ._ext import ext, status_word
from .rope import AxisRope


class PackedPages(NamedTuple):
    """K or V pages of one layer in 8 bits: ``codes`` float8_e4m3fn ``[pages, page_size, kv_heads, head_dim]`` and ``scales``
    float8_e8m0fnu ``[kv_heads, pages, page_size]``; head_dim 64 or 128.

    A row (one token's channels of one KV head) holds ``code * scale``, the scale the smallest power of two that brings the row's
    largest magnitude to 448 and below, within 2^-124 .. 2^119 (bf16) or 2^-15 .. 2^7 (fp16, whose numbers above 57,344 are
    held as that): so what a row holds is a number of the 16-bit type that it came in, off by half a step of e4m3 (2^-4 of its size, or
    2^-10 of the scale where that is more), and reading rounds nothing. A row with a NaN or infinity has a scale of NaN and reads as NaN."""

    codes: torch.Tensor
    scales: torch.Tensor

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, device) -> "PackedPages":
        """Pages that hold zeros."""
        codes = torch.zeros(pages, page_size, kv_heads, head_dim, dtype=torch.uint8, device=device)
        scales = torch.full((kv_heads, pages, page_size), 127, dtype=torch.uint8, device=device)
        return cls(codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu))


def _parts(pages):
    """Tensor of pages, and its scales where they are packed."""
    return pages if type(pages) is PackedPages else (pages, None)


def _both(k_pages, v_pages) -> bool:
    """Whether the pages are packed (both or neither)."""
    packed = type(k_pages) is PackedPages
    if packed is not (type(v_pages) is PackedPages):
        raise ConfigurationError("both or neither of k_pages and v_pages must be packed")
    return packed


def append(q, k, v, positions, rope: AxisRope, k_pages, v_pages, block_table, kv_lens, cu_q, *, out=None):
    """Rotate ``q[T, heads, D]`` and ``k[T, kv_heads, D]`` at ``positions[T, axes]`` and write ``k`` and ``v`` into
    their sequences' pages, in one launch. Returns the rotated ``q`` (``out`` if given). bf16 or fp16; into packed pages ``k``
    and ``v`` are quantised from the rotated rows in FP32, in one rounding."""
    if not q.is_cuda:
        raise UnsupportedError("append needs CUDA tensors")
    if q.size(-1) != rope.head_dim:
        raise ConfigurationError(f"the rotation is for head_dim {rope.head_dim}, q has {q.size(-1)}")
    device = q.device
    if _both(k_pages, v_pages):
        return ext().packed_append(q, k, v, positions, rope.plan(device), *k_pages, *v_pages, block_table, kv_lens, cu_q, out,
                                   status_word(device))
    return ext().paged_append(q, k, v, positions, rope.plan(device), k_pages, v_pages, block_table, kv_lens, cu_q, out,
                              status_word(device))


def store(k, v, k_pages: PackedPages, v_pages: PackedPages, block_table, kv_lens, cu_q):
    """Write ``k`` and ``v[T, kv_heads, D]`` (bf16 or fp16) as they are into their sequences' packed pages, in one launch."""
    if not k.is_cuda:
        raise UnsupportedError("store needs CUDA tensors")
    if not _both(k_pages, v_pages):
        raise ConfigurationError("store writes packed pages")
    ext().packed_store(k, v, *k_pages, *v_pages, block_table, kv_lens, cu_q, status_word(k.device))


def read(k_pages: PackedPages, v_pages: PackedPages, block_table, starts, rows: int, *, dtype=torch.bfloat16):
    """K and V of sequences out of packed pages, dense ``[rows, kv_heads, D]`` in the 16-bit type that they were written from: the first
    ``starts[s + 1] - starts[s]`` tokens of sequence ``s`` are rows ``starts[s]`` and on (``starts [seqs + 1]`` int32 on the device).
    Rows of no sequence hold anything."""
    if not _both(k_pages, v_pages):
        raise ConfigurationError("read takes packed pages")
    if not k_pages.codes.is_cuda:
        raise UnsupportedError("read needs CUDA tensors")
    return ext().packed_read(*k_pages, *v_pages, block_table, starts, rows, dtype, status_word(k_pages.codes.device))


def attention(q, k_pages, v_pages, block_table, kv_lens, cu_q, *, max_q_len: int, causal: bool = False,
              window: int | None = None, sinks: int = 0, scale: float | None = None, return_lse: bool = False, out=None):
    """``softmax(scale * q k^T) v`` of every sequence's new tokens ``q[T, heads, D]`` over its pages; heads in groups of
    ``heads / kv_heads`` share a KV head. bf16 or fp16, head_dim 64 or 128. Scores, maxima, sums and outputs are FP32; the
    probabilities are rounded to the inputs' type for the product with ``v`` (their sum is not), as the tensor core takes
    them: against 64 bits the error of a bf16 chunk grows from 0.0017 to 0.0022 of the output's size by it.

    ``causal``: a token sees positions up to its own; else every new token sees the whole sequence (a chunk that is
    bidirectional in itself). ``window`` keeps the last ``window`` of the positions it would see, and the first
    ``sinks`` of the sequence. A token that sees nothing gets zeros (and ``lse`` of minus infinity). A
    score of NaN makes its token's output and ``lse`` NaN; one of plus infinity makes ``lse`` plus infinity, the output NaN.
    Rows of ``v`` that no new token of the sequence sees may hold anything; one with a NaN or infinity that some see may make
    the outputs of tokens beside them NaN too (a weight of zero times NaN).
    ``max_q_len`` bounds the new tokens of every sequence (more are reported, see the module). Rows of ``q`` outside of
    ``cu_q`` belong to no sequence: they have no result (a new output holds anything there). ``return_lse`` adds the natural log-sum-exp ``[T, heads]``.

    ``block_table`` may be ``[seqs, kv_heads, width]``, a table for each KV head. Packed pages give what their rows read as
    :func:`read` gives, in ``q``'s type, which must be the one that the rows were written from (fp16 does not hold what bf16's
    range of scales does). With up to 48 rows (new tokens x heads of a group) the codes are taken as they are and the
    probabilities times V's scales are rounded to fp16 (a key's by half a step, or by 2^-32 of the largest where that is more);
    channels of ``q`` below 2^-20 of their row's largest are off by up to 2^-31 of that.
    With more, the pages that are seen are expanded first: 16-bit copies of them for the time of the call, in room for as many
    pages as the table has entries, or a window leaves of them, or the pool has; in a batch with one long prompt among single
    tokens, of all its sequences."""
    if not q.is_cuda:
        raise UnsupportedError("paged attention needs CUDA tensors")
    if window is not None and window < 1:
        raise ConfigurationError(f"window {window} must be positive")
    k_scales = v_scales = None
    if _both(k_pages, v_pages):
        (k_pages, k_scales), (v_pages, v_scales) = k_pages, v_pages
    out, lse = ext().paged_attention(q, k_pages, v_pages, block_table, kv_lens, cu_q, max_q_len, causal, window or 0, sinks,
                                     scale, return_lse, out, status_word(q.device), k_scales, v_scales)
    return (out, lse) if return_lse else out


def attention_form(tokens, heads, kv_heads, head_dim, seqs, width, page_size, *, max_q_len: int, causal: bool = False,
                   window: int | None = None, sinks: int = 0, packed: bool = False, tables: bool = False, device: int = 0) -> str:
    """Which form of the kernels a call of :func:`attention` with these sizes takes: ``"few rows, cluster N"``, ``"few rows,
    line"``, ``"twin N"``, ``"direct N"`` (``N`` CTAs to a cluster) or ``"planned"``. ``width``: columns of the block table.
    ``packed``: over packed pages, ``"few rows, ..."``, ``"S slices, ..."`` (of 16 rows) or ``"expanded, "`` and a form of more rows.
    ``tables``: with a table for each KV head, also ``"twin 1, then M items in N"`` (the last ``M`` in clusters of ``N``)."""
    return ext().paged_attention_form(device, tokens, heads, kv_heads, head_dim, seqs, width, page_size, max_q_len, causal,
                                      window or 0, sinks, packed, tables)


def blocks(pages, block: int):
    """Pages ``[pages, page_size, kv_heads, D]`` (or packed ones) cut into pages of ``block`` tokens, a view: page ``p`` becomes pages
    ``p * page_size / block`` and on. ``block`` divides the page size and is a multiple of 8; where it is less, the pages must lie one
    after the other."""
    tensor, scales = _parts(pages)
    (count, size, heads, dim), (page, token, *rest) = tensor.shape, tensor.stride()
    if block < 8 or block % 8 or size % block:
        raise ConfigurationError(f"blocks of {block} tokens must be multiples of 8 and divide the page size, {size}")
    if block == size:
        return pages
    if count > 1 and page != size * token or scales is not None and count > 1 and scales.stride(1) != size:
        raise ConfigurationError("pages that are cut into blocks must lie one after the other")
    number = count * (size // block)
    tensor = tensor.as_strided((number, block, heads, dim), (block * token, token, *rest))
    if scales is None:
        return tensor
    return PackedPages(tensor, scales.as_strided((heads, number, block), (scales.stride(0), block, 1)))


def block_means(k_pages, means, block_table, kv_lens, cu_q, *, max_q_len: int):
    """Bring the means of the keys of blocks up to date after new tokens were written: those of the blocks that hold the last
    ``cu_q[s + 1] - cu_q[s]`` tokens of every sequence, over the tokens that they hold. ``means [pages, page_size / block,
    kv_heads, D]`` of the pages' type (of packed pages bf16 or fp16) lie beside the pages. Sums are in FP64."""
    tensor, scales = _parts(k_pages)
    if not tensor.is_cuda:
        raise UnsupportedError("block_means needs CUDA tensors")
    ext().paged_block_means(tensor, scales, means, block_table, kv_lens, cu_q, max_q_len, status_word(tensor.device))
    return means


class ChosenBlocks(NamedTuple):
    """A batch for :func:`attention` over :func:`blocks`: every query block is a sequence of its own. ``table [items, kv_heads,
    width]`` (-1 behind the chosen blocks), ``kv_lens [items]``, ``cu_q [items + 1]``; ``max_q_len`` new tokens at most."""

    table: torch.Tensor
    kv_lens: torch.Tensor
    cu_q: torch.Tensor
    max_q_len: int


def select_blocks(q, means, block_table, kv_lens, cu_q, *, block: int, keep: int, max_q_len: int, query_block: int = 1,
                  causal: bool = False, sinks: int = 0, recent: int = 0) -> ChosenBlocks:
    """Choose the blocks of ``block`` positions that the new tokens ``q[T, heads, D]`` attend to, for every ``query_block`` of them
    (consecutive tokens of a sequence; 1: each its own) and KV head: the ``keep`` blocks of the past that score highest, and always those that
    hold the first ``sinks`` positions, the ``recent`` positions before the new tokens, and the new tokens; with ``causal`` the
    ``recent`` positions before the query block, and the query block (new tokens before those are past like any). The tokens of a query block share a choice that all of their queries make: ``causal`` keeps each
    from seeing later positions, but which blocks of the past it sees depends on the queries of the tokens after it in its query block.
    A prompt read in query blocks is thus not the same as its tokens one by one (``query_block=1`` is).

    A block's score is the largest over the heads of the group of the sum of the query block's ``q`` times the mean of the
    block's keys (``means`` from :func:`block_means`), in FP64: the choice does not depend on the order of sums. Equal scores go to the lower block; a
    score of NaN comes last. A table has at most 12,288 blocks (its width times the blocks of a page), fewer where groups are large:
    16 bytes a block and about ``16 D + 260`` a head of a group must fit 224 KB (11 heads of 128 with 12,288 blocks, 88 with
    1,024); other calls are refused. Attention over the choice (its tables name the past in order, the query block's own tokens
    last, so that ``causal`` holds there)::

        chosen = select_blocks(q, means, block_table, kv_lens, cu_q, block=64, keep=16, max_q_len=n, causal=True)
        out = attention(q, blocks(k_pages, 64), blocks(v_pages, 64), chosen.table, chosen.kv_lens, chosen.cu_q,
                        max_q_len=chosen.max_q_len, causal=True)
    """
    if not q.is_cuda:
        raise UnsupportedError("the choice of blocks needs CUDA tensors")
    table, lens, cu = ext().paged_select_blocks(q, means, block_table, kv_lens, cu_q, block, keep, query_block, max_q_len, causal,
                                                sinks, recent, status_word(q.device))
    return ChosenBlocks(table, lens, cu, min(query_block, max_q_len))


def copy_pages(storage, source, target, rows=None):
    """Copy pages ``source[i]`` to ``target[i]`` (int32 vectors) in every plane of ``storage [planes, pages, page_size,
    ...]``: whole pages, or their first ``rows[i]`` tokens. Pairs of -1 are skipped. Targets must differ from one another
    and from every source (the copies run at the same time)."""
    if not storage.is_cuda:
        raise UnsupportedError("copy_pages needs CUDA tensors")
    ext().pages_copy(storage, source, target, rows, status_word(storage.device))
    return storage


class PageTable:
    """The page table of ``seqs`` sequence slots over ``pages`` pages, one int32 tensor ``state`` on the device:
    ``refcount [pages]``, ``lens [seqs]`` and ``block_table [seqs, width]`` are its parts (views).

    All operators run on the device in stream order and take int32 vectors on it. Free pages are taken lowest first, in
    the order of the call's sequences. A call that cannot be served changes nothing (see the module)."""

    def __init__(self, state: torch.Tensor, *, pages: int, seqs: int, page_size: int):
        cells = state.numel() - pages - seqs
        if state.dim() != 1 or state.dtype is not torch.int32 or pages < 1 or seqs < 1 or cells < 1 or cells % seqs:
            raise ConfigurationError(f"a page table of {pages} pages and {seqs} sequences is an int32 vector of pages + "
                                     f"seqs + seqs * width entries, got {state.dtype} {tuple(state.shape)}")
        self.state, self.pages, self.seqs, self.page_size = state, pages, seqs, page_size

    @property
    def refcount(self) -> torch.Tensor:
        """``[pages]``: sequences that hold each page (0: it is free)."""
        return self.state[:self.pages]

    @property
    def lens(self) -> torch.Tensor:
        """``[seqs]``: tokens that each sequence holds."""
        return self.state[self.pages:self.pages + self.seqs]

    @property
    def block_table(self) -> torch.Tensor:
        """``[seqs, width]``: page of each block of each sequence, -1 for none."""
        return self.state[self.pages + self.seqs:].view(self.seqs, -1)

    @classmethod
    def empty(cls, pages: int, seqs: int, width: int, page_size: int, device) -> "PageTable":
        """All pages free, no sequence holding any; ``width`` blocks per sequence at most."""
        state = torch.zeros(pages + seqs + seqs * width, dtype=torch.int32, device=device)
        state[pages + seqs:] = -1
        return cls(state, pages=pages, seqs=seqs, page_size=page_size)

    def _parts(self):
        return self.state, self.pages, self.seqs, self.page_size

    def allocate(self, seqs, lens):
        """Sequences ``seqs[i]`` grow to ``lens[i]`` tokens (at least what they hold)."""
        ext().pages_allocate(*self._parts(), seqs, lens, status_word(self.state.device))

    def fork(self, parents, children, lens, storage, sides=()):
        """Sequences ``children[i]`` (holding nothing) take the first ``lens[i]`` tokens of ``parents[i]``: whole pages
        are shared, the rows of a partly filled last page are copied in every plane of ``storage [planes, pages,
        page_size, ...]`` to a page of the child's own, and with them its page in ``sides`` (up to two tensors ``[planes, pages,
        ...]``: scales of packed pages, means of blocks)."""
        ext().pages_fork(*self._parts(), parents, children, lens, storage, status_word(self.state.device), list(sides))

    def release(self, seqs):
        """Sequences ``seqs[i]`` give all their pages back; a page is free when no sequence holds it."""
        ext().pages_release(*self._parts(), seqs, status_word(self.state.device))

    def compact(self, storage, sides=()) -> torch.Tensor:
        """Move the pages in use to the front of ``storage`` (and of ``sides``) and follow them in the tables. Returns their
        number, an int32 tensor of one entry on the device."""
        return ext().pages_compact(*self._parts(), storage, status_word(self.state.device), list(sides))
