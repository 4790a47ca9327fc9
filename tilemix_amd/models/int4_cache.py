"""A transformers KV cache in 4 bits (``tilemix_amd.attention.hip.paged_int4``) for the TileMix models.

``Int4KVCache`` holds the K and V of every layer in pages of 4-bit codes, which all layers place by one
set of page tables.  Passed as ``past_key_values``

* the TileMix attention modules prefill from the K and V at hand, as with any cache, and store them; later
  tokens -- a decode step, drafts, the next chunk of a prompt, of any length -- attend to the cache
  itself;
* any other attention gets from ``update`` what it expects of a cache, the K and V of all tokens (the
  stored ones read back).

A padded batch needs its attention mask, which the kernels do not read: with a mask the modules
take the second way, unless the cache was made with ``unpadded=True`` (the promise that no
sequence is padded; transformers builds a causal mask for several new tokens even then).
"""
from __future__ import annotations

import torch
from torch import Tensor
from transformers.cache_utils import Cache, CacheLayerMixin

from ..attention.hip.paged_int4 import PagedInt4Cache, PageTables, load_int4, paged_int4_attention, store_int4

__all__ = ["Int4KVCache"]


def _rows(x: Tensor) -> Tensor:
    """[B, H, T, D] as token-major rows [B T, H, D] (a view where the layout allows one)."""
    b, h, t, d = x.shape
    return x.transpose(1, 2).reshape(b * t, h, d)


class _Int4Layer(CacheLayerMixin):
    is_sliding = False

    def __init__(self, owner: "Int4KVCache", pool: PagedInt4Cache, idx: int):
        super().__init__()
        self.owner, self.pool, self.idx, self.seen = owner, pool, idx, 0
        self.is_initialized = True

    def lazy_initialization(self, *args, **kwargs) -> None:
        return None

    def update(self, key_states, value_states, *args, **kwargs):
        return self.owner._update(self, key_states, value_states)

    def get_seq_length(self, *args, **kwargs) -> int:
        return self.seen

    def get_mask_sizes(self, query_length, *args, **kwargs) -> tuple[int, int]:
        # (a tensor of positions instead of their number in transformers 4.x)
        new = query_length.shape[0] if isinstance(query_length, Tensor) else query_length
        return self.seen + new, 0

    def get_max_length(self) -> int:
        return self.owner.max_tokens

    get_max_cache_shape = get_max_length

    def reset(self) -> None:
        self.owner._keep(0)

    def _unsupported(self, *args, **kwargs):
        raise NotImplementedError("Int4KVCache neither moves, reorders nor repeats its sequences")

    offload = prefetch = reorder_cache = batch_repeat_interleave = batch_select_indices = _unsupported


class Int4KVCache(Cache):
    """Room for ``max_tokens`` tokens of ``batch`` sequences in each of ``layers`` layers."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, batch: int, max_tokens: int, *, page_size: int = 64,
                 device="cuda", unpadded: bool = False):
        if min(layers, batch, max_tokens, page_size) < 1:
            raise ValueError(f"Int4KVCache needs layers, sequences, tokens and a page size of at least 1, got {layers}, "
                             f"{batch}, {max_tokens}, {page_size}")
        columns = -(-max_tokens // page_size)
        pools = (PagedInt4Cache.empty(batch * columns, kv_heads, head_dim, page_size, device) for _ in range(layers))
        super().__init__(layers=[_Int4Layer(self, pool, idx) for idx, pool in enumerate(pools)])
        self.tables = PageTables.empty(batch * columns, batch, columns, page_size, device)
        self.batch, self.max_tokens, self.unpadded = batch, max_tokens, unpadded
        self.length = 0  # tokens of each sequence that the tables have a place for
        self._plan = self._new = None

    @classmethod
    def for_model(cls, model, batch: int, max_tokens: int, **kwargs) -> "Int4KVCache":
        c = model.config
        head_dim = getattr(c, "head_dim", None) or c.hidden_size // c.num_attention_heads
        kwargs.setdefault("device", model.device)
        return cls(c.num_hidden_layers, c.num_key_value_heads, head_dim, batch, max_tokens, **kwargs)

    def serves(self, attention_mask) -> bool:
        """Whether attention over the cache itself gives what the mask asks for."""
        return self.unpadded or attention_mask is None

    def append(self, key_states: Tensor, value_states: Tensor, layer_idx: int) -> None:
        """Store the new tokens' K and V [B, H, T, D] of a layer.  The layers of a model take turns with the same
        tokens; the first one gets them their places."""
        layer = self.layers[layer_idx]
        batch, _, new, _ = key_states.shape
        if batch != self.batch:
            raise ValueError(f"Int4KVCache holds {self.batch} sequences, got {batch}")
        if layer.seen == self.length:
            if key_states.is_cuda and torch.cuda.is_current_stream_capturing():
                # The lengths that bound the kernels' work are kept here: a replay would go on with the captured ones.
                raise RuntimeError("Int4KVCache counts its tokens on the host and takes no part in a graph capture; "
                                   "PageTables and paged_int4_attention do")
            if self.length + new > self.max_tokens:
                raise ValueError(f"Int4KVCache has room for {self.max_tokens} tokens a sequence, "
                                 f"got {self.length} and {new} more")
            if self._new is None or self._new[0] != new:
                self._new = new, torch.full((batch,), new, dtype=torch.int32, device=self.tables.seq_lens.device)
            self._plan = self.tables.extend(self._new[1], batch * new)
            self.length += new
        elif layer.seen + new != self.length:
            raise ValueError(f"layer {layer_idx} got {new} tokens after {layer.seen}, the first layer holds {self.length}")
        store_int4(_rows(key_states), _rows(value_states), layer.pool, self._plan.slots)
        layer.seen += new

    def attend(self, query_states: Tensor, layer_idx: int, scale: float) -> Tensor:
        """Causal attention of the last T tokens' queries [B, H, T, D] over a layer's tokens: [B, T, H, D]."""
        layer = self.layers[layer_idx]
        b, h, t, d = query_states.shape
        out = paged_int4_attention(_rows(query_states), layer.pool, self.tables.block_table, self.tables.seq_lens, None, t,
                                   layer.seen, sm_scale=scale)
        return out.view(b, t, h, d)

    def _update(self, layer: _Int4Layer, key_states: Tensor, value_states: Tensor):
        first = layer.seen == 0
        self.append(key_states, value_states, layer.idx)
        if first:
            return key_states, value_states
        tokens = layer.seen
        ends = torch.arange(0, (self.batch + 1) * tokens, tokens, dtype=torch.int32, device=key_states.device)
        both = load_int4(layer.pool, self.tables.block_table, ends, self.batch * tokens, dtype=key_states.dtype)
        return tuple(x.view(self.batch, tokens, *x.shape[1:]).transpose(1, 2) for x in both)

    def _keep(self, tokens: int) -> None:
        if tokens < self.length:
            self.tables.truncate(torch.full_like(self.tables.seq_lens, tokens))
            self.length = tokens
        for layer in self.layers:
            layer.seen = min(layer.seen, tokens)

    def crop(self, tokens_to_remove: int) -> None:
        """Drop the last ``-tokens_to_remove`` tokens; a positive number is how many stay (as in transformers)."""
        self._keep(max(0, tokens_to_remove if tokens_to_remove > 0 else self.length + tokens_to_remove))

    def reset(self) -> None:
        self._keep(0)
