"""A paged 4-bit KV cache and the attention that decodes and continues prompts over it.

The prefill attention of ``tilemix.py`` reads fp16 K and V; this module is what comes after it
(the reference stops at the prefill: below 16 query tokens it runs the model's own attention over
an fp16 cache, models/tilemix_llama.py:527-537).

* ``PagedInt4Cache`` -- K and V of one layer in pages of 4-bit codes;
* ``PageTables`` -- which pages each sequence owns, kept and changed on the GPU;
* ``store_int4`` -- new K and V rows into their slots;
* ``load_int4`` -- sequences back as fp16 or bf16 rows;
* ``paged_int4_attention`` -- packed queries against the cache.

Format.  A (token, KV head) row of ``head_dim`` (1 to 128) values is split into groups of 32
channels.  A group holds a scale s and a minimum m in fp16 and a 4-bit code n a channel, and
stands for the values fp16(n s + m), with m = fp16(min x), s = fp16((max x - min x) / 15) and n =
rint((x - m) / s) in 0 .. 15 (x clamped to +-65408; a NaN makes its group NaN).  At head_dim
128 that is 80 bytes a row instead of 256.

Every call is asynchronous on the current stream, reads nothing back to the host, may be captured
into a graph, and returns tensors without an autograd graph.  What it does not take raises
``TypeError`` or ``ValueError`` before any launch; there is no CPU path (``RuntimeError``).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch import Tensor

from ... import _native

GROUP = 32


def _width(head_dim: int) -> int:
    return -(-head_dim // GROUP) * GROUP


class PagedInt4Cache:
    """K and V of one layer: ``codes`` uint8 [pages, heads, page_size, width / 2] (channel 2j in the
    low half of byte j; width is head_dim rounded up to 32) and ``params`` fp16
    [pages, heads, page_size, width / 32, 2] (scale, minimum), contiguous.  page_size is a multiple of 16."""

    __slots__ = ("_args",)

    def __init__(self, k_codes: Tensor, k_params: Tensor, v_codes: Tensor, v_params: Tensor, head_dim: int):
        _native.host().kv4_check(k_codes, k_params, v_codes, v_params, head_dim)
        self._args = (k_codes, k_params, v_codes, v_params, head_dim)

    k_codes = property(lambda self: self._args[0])
    k_params = property(lambda self: self._args[1])
    v_codes = property(lambda self: self._args[2])
    v_params = property(lambda self: self._args[3])
    head_dim = property(lambda self: self._args[4])

    @classmethod
    def empty(cls, pages: int, heads: int, head_dim: int, page_size: int = 64, device="cuda") -> "PagedInt4Cache":
        """A cache whose rows are undefined until they are stored."""
        shape, width = (pages, heads, page_size), _width(head_dim)
        codes = (torch.empty((*shape, width // 2), dtype=torch.uint8, device=device) for _ in range(2))
        params = (torch.empty((*shape, width // GROUP, 2), dtype=torch.float16, device=device) for _ in range(2))
        return cls(next(codes), next(params), next(codes), next(params), head_dim)

    @property
    def pages(self) -> int:
        return self.k_codes.shape[0]

    @property
    def heads(self) -> int:
        return self.k_codes.shape[1]

    @property
    def page_size(self) -> int:
        return self.k_codes.shape[2]


class SlotPlan(NamedTuple):
    """Where the new tokens of a step go (``PageTables.extend``)."""

    slots: Tensor       # int64 [num_tokens]: page * page_size + row; -1: none
    positions: Tensor   # int64 [num_tokens]: place in the sequence; 0 where there is no slot
    cu_seqlens: Tensor  # int32 [sequences + 1]: each sequence's new tokens
    granted: Tensor     # int32 [sequences]: 1 where the sequence got its tokens


class PageTables:
    """The pages and lengths of up to 4096 sequences and the stack of free pages, on the GPU:
    ``block_table`` int32 [sequences, columns], ``seq_lens`` int32 [sequences], ``free_pages`` int32
    [pages], of which the first ``free_count`` (int32 [1]) are free.  The calls change these tensors
    in place, in the order of the stream they run on: calls on several streams have to be ordered by
    the caller.  One ``PageTables`` serves the caches of all layers."""

    __slots__ = ("_args", "page_size")

    def __init__(self, block_table: Tensor, seq_lens: Tensor, free_pages: Tensor, free_count: Tensor, page_size: int):
        ticket = torch.zeros(1, dtype=torch.int32, device=block_table.device)
        self._args, self.page_size = (block_table, seq_lens, free_pages, free_count, ticket), page_size

    block_table = property(lambda self: self._args[0])
    seq_lens = property(lambda self: self._args[1])
    free_pages = property(lambda self: self._args[2])
    free_count = property(lambda self: self._args[3])

    @classmethod
    def empty(cls, pages: int, sequences: int, columns: int, page_size: int = 64, device="cuda") -> "PageTables":
        """All pages free, page 0 on top of the stack; no sequence holds a token."""
        return cls(torch.full((sequences, columns), -1, dtype=torch.int32, device=device),
                   torch.zeros(sequences, dtype=torch.int32, device=device),
                   torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device),
                   torch.full((1,), pages, dtype=torch.int32, device=device), page_size)

    def extend(self, new_lens: Tensor, num_tokens: int) -> SlotPlan:
        """Give sequence b ``new_lens[b]`` (int32) more tokens; ``num_tokens``: entries of the plan, at
        least the sum of new_lens.

        A sequence is granted its tokens if they fit its table row and ``num_tokens`` and the
        pages that it and the sequences before it need are free (or it needs none); one that is not
        keeps its length and pages, its entries of the plan have slot -1 and position 0, and its
        place in ``cu_seqlens`` stays."""
        return SlotPlan(*_native.host().kv4_extend(*self._args, new_lens, self.page_size, num_tokens))

    def truncate(self, lens: Tensor) -> None:
        """Sequence b keeps its first ``min(seq_lens[b], lens[b])`` tokens (0: it is done).  Pages that
        are no longer needed go back to the stack in the opposite order of ``extend``, so that
        truncating to the lengths before an extension undoes it."""
        _native.host().kv4_truncate(*self._args, lens, self.page_size)


def store_int4(k: Tensor, v: Tensor, cache: PagedInt4Cache, slots: Tensor) -> None:
    """Quantise row t of k and v [tokens, heads, head_dim] (fp16 or bf16, any strides) into slot
    ``slots[t]`` (int64).  A slot outside the cache is skipped.  The slots of a call must differ: of
    two rows with one slot a mixture may remain."""
    _native.host().kv4_store(*cache._args, k, v, slots)


def load_int4(cache: PagedInt4Cache, block_table: Tensor, cu_seqlens: Tensor, num_tokens: int,
              dtype: torch.dtype = torch.float16) -> tuple[Tensor, Tensor]:
    """Sequences as packed rows: (k, v) [num_tokens, heads, head_dim], the first ``cu_seqlens[b + 1] -
    cu_seqlens[b]`` tokens of sequence b from row ``cu_seqlens[b]`` on -- the K and V of
    ``tilemix_attention_with_quant``.  Rows of no sequence, or of a page that the table does not name,
    are zeros."""
    return _native.host().kv4_load(*cache._args, block_table, cu_seqlens, num_tokens, dtype)


def paged_int4_attention(q: Tensor, cache: PagedInt4Cache, block_table: Tensor, seq_lens: Tensor,
                         cu_seqlens_q: Optional[Tensor], max_seqlen_q: int, max_seqlen_k: int, *,
                         causal: bool = True, sm_scale: Optional[float] = None,
                         out: Optional[Tensor] = None) -> Tensor:
    """softmax(sm_scale q k^T) v of packed queries q [tokens, query heads, head_dim] (fp16 or bf16) over
    the cache, in q's type; sm_scale defaults to head_dim ** -0.5.

    Sequence b has ``seq_lens[b]`` keys, its queries are ``cu_seqlens_q[b] .. cu_seqlens_q[b + 1] - 1``
    (None: max_seqlen_q of each sequence) and are its last tokens: with ``causal`` query i of nq sees
    the keys up to ``seq_lens[b] - nq + i``, without it all of them.  Query head h reads KV head
    ``h // (query heads // KV heads)``.  A query that sees no key gets zeros; keys of a page that the
    table does not name are not seen.  ``max_seqlen_q`` and ``max_seqlen_k`` (and the places of a table
    row) bound the queries and keys of a sequence: a longer one counts as that long.  Rows behind the
    last query are left as they were in ``out`` (undefined without one), which may be q itself."""
    return _native.host().kv4_attention(*cache._args, q, block_table, seq_lens, cu_seqlens_q, max_seqlen_q,
                                        max_seqlen_k, causal, sm_scale, out)
