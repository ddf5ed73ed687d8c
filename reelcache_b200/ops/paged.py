"""A paged KV cache's operators on sm_100a: writing new tokens (csrc/paged/rotate.cu), attending over the pages
(attend_short.cu, attend_chunk.cu) and the page table (table.cu).

Pages: ``k_pages, v_pages [pages, page_size, kv_heads, head_dim]`` of one layer (any 16-byte aligned strides; the page
size is a multiple of 8 tokens). A batch of sequences is described by ``block_table [seqs, width]`` (page of each block
of ``page_size`` tokens, -1 for none), ``kv_lens [seqs]`` (tokens held, the new ones included) and ``cu_q [seqs + 1]``
(where each sequence's new tokens begin in ``q``), all int32 on the device (rows of the table may be strided: a slice
``table[:, :n]`` will do): nothing is read back, every call can be captured in a graph. Sequence ``s``'s new tokens are
its last ``cu_q[s + 1] - cu_q[s]`` positions.

Calls with page numbers outside the pool, lengths that do not fit their tensors or bounds, or page-table calls that cannot
be served, do nothing out of bounds and are reported by :func:`reelcache_b200.ops._ext.check_status`.
"""

from __future__ import annotations

import torch

from ..errors import ConfigurationError, UnsupportedError
from ._ext import ext, status_word
from .rope import AxisRope


def append(q, k, v, positions, rope: AxisRope, k_pages, v_pages, block_table, kv_lens, cu_q, *, out=None):
    """Rotate ``q[T, heads, D]`` and ``k[T, kv_heads, D]`` at ``positions[T, axes]`` and write ``k`` and ``v`` into
    their sequences' pages, in one launch. Returns the rotated ``q`` (``out`` if given). bf16 or fp16."""
    if not q.is_cuda:
        raise UnsupportedError("append needs CUDA tensors")
    if q.shape[-1] != rope.head_dim:
        raise ConfigurationError(f"the rotation is for head_dim {rope.head_dim}, q has {q.shape[-1]}")
    device = q.device
    return ext().paged_append(q, k, v, positions, rope.plan(device), k_pages, v_pages, block_table, kv_lens, cu_q, out,
                              status_word(device))


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
    ``cu_q`` belong to no sequence: they have no result (a new output holds anything there). ``return_lse`` adds the natural log-sum-exp ``[T, heads]``."""
    if not q.is_cuda:
        raise UnsupportedError("paged attention needs CUDA tensors")
    if window is not None and window < 1:
        raise ConfigurationError(f"window {window} must be positive")
    out, lse = ext().paged_attention(q, k_pages, v_pages, block_table, kv_lens, cu_q, max_q_len, causal, window or 0, sinks,
                                     scale, return_lse, out, status_word(q.device))
    return (out, lse) if return_lse else out


def attention_form(tokens, heads, kv_heads, head_dim, seqs, width, page_size, *, max_q_len: int, causal: bool = False,
                   window: int | None = None, sinks: int = 0, device: int = 0) -> str:
    """Which form of the kernels a call of :func:`attention` with these sizes takes: ``"few rows, cluster N"``, ``"few rows,
    line"``, ``"twin N"``, ``"direct N"`` (``N`` CTAs to a cluster) or ``"planned"``. ``width``: columns of the block table."""
    return ext().paged_attention_form(device, tokens, heads, kv_heads, head_dim, seqs, width, page_size, max_q_len, causal,
                                      window or 0, sinks)


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

    def fork(self, parents, children, lens, storage):
        """Sequences ``children[i]`` (holding nothing) take the first ``lens[i]`` tokens of ``parents[i]``: whole pages
        are shared, the rows of a partly filled last page are copied in every plane of ``storage [planes, pages,
        page_size, ...]`` to a page of the child's own."""
        ext().pages_fork(*self._parts(), parents, children, lens, storage, status_word(self.state.device))

    def release(self, seqs):
        """Sequences ``seqs[i]`` give all their pages back; a page is free when no sequence holds it."""
        ext().pages_release(*self._parts(), seqs, status_word(self.state.device))

    def compact(self, storage) -> torch.Tensor:
        """Move the pages in use to the front of ``storage`` and follow them in the tables. Returns their number, an
        int32 tensor of one entry on the device."""
        return ext().pages_compact(*self._parts(), storage, status_word(self.state.device))
