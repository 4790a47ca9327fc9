"""CPU tests of the 4-bit transformers cache: bookkeeping, refusals and the way that an attention
module's call takes.  What it computes is in test_gpu_int4_cache.py."""
from __future__ import annotations

import pytest
import torch
from transformers import DynamicCache, LlamaConfig, LlamaForCausalLM

from tilemix_amd.models import tilemix_llama as TL
from tilemix_amd.models._common import int4_route
from tilemix_amd.models.int4_cache import Int4KVCache


def make(**kw):
    args = dict(layers=2, kv_heads=2, head_dim=64, batch=3, max_tokens=40, page_size=16, device="cpu")
    args.update(kw)
    return Int4KVCache(args.pop("layers"), args.pop("kv_heads"), args.pop("head_dim"), args.pop("batch"),
                       args.pop("max_tokens"), **args)


def kv(batch=3, tokens=4, heads=2, dim=64):
    return torch.zeros(batch, heads, tokens, dim, dtype=torch.float16)


def test_shapes_and_lengths():
    c = make()
    assert len(c) == 2 and c.get_seq_length() == 0 and c.get_max_length() == 40 and c.layers[1].get_max_cache_shape() == 40
    assert c.layers[0].pool.pages == 9 and tuple(c.tables.block_table.shape) == (3, 3)
    assert c.get_mask_sizes(5, 1) == (5, 0) and c.layers[0].get_mask_sizes(torch.arange(7)) == (7, 0)
    cfg = LlamaConfig(vocab_size=96, hidden_size=128, intermediate_size=256, num_hidden_layers=3, num_attention_heads=4,
                      num_key_value_heads=2)
    m = Int4KVCache.for_model(LlamaForCausalLM(cfg), 2, 100)
    assert len(m) == 3 and m.layers[0].pool.heads == 2 and m.layers[0].pool.head_dim == 32
    assert m.layers[0].pool.k_codes.device.type == "cpu"


def test_refusals():
    c = make()
    with pytest.raises(ValueError, match="holds 3 sequences, got 2"):
        c.append(kv(batch=2), kv(batch=2), 0)
    with pytest.raises(ValueError, match="room for 40 tokens"):
        c.update(kv(tokens=41), kv(tokens=41), 0)
    c.length = c.layers[0].seen = 30  # (as after 30 tokens in the first layer)
    with pytest.raises(ValueError, match="room for 40 tokens"):
        c.append(kv(tokens=11), kv(tokens=11), 0)
    with pytest.raises(ValueError, match="layer 1 got 7 tokens after 0"):
        c.append(kv(tokens=7), kv(tokens=7), 1)
    with pytest.raises(RuntimeError, match="GPU"):
        make().update(kv(), kv(), 0)
    for call in (lambda l: l.reorder_cache(torch.tensor([0, 1, 2])), lambda l: l.batch_repeat_interleave(2),
                 lambda l: l.batch_select_indices(torch.tensor([0])), lambda l: l.offload()):
        with pytest.raises(NotImplementedError):
            call(c.layers[0])
    with pytest.raises(ValueError, match="head_dim"):
        make(head_dim=256)


def test_route():
    """(over the cache, parent): without the cache as before; with it by tokens seen and mask."""
    mask = torch.zeros(1, 1, 4, 4)
    for past in (None, DynamicCache()):
        assert int4_route(past, 0, None, 15) == (False, True) and int4_route(past, 0, mask, 16) == (False, False)
    c = make()
    assert int4_route(c, 0, None, 16) == (False, False) and int4_route(c, 0, mask, 16) == (False, False)
    assert int4_route(c, 0, None, 15) == (True, False) and int4_route(c, 0, mask, 15) == (False, True)
    c.layers[0].seen = 5
    assert int4_route(c, 0, None, 200) == (True, False) and int4_route(c, 0, mask, 200) == (False, True)
    assert int4_route(c, 1, mask, 200) == (False, False)
    c.unpadded = True
    assert int4_route(c, 0, mask, 1) == (True, False) and int4_route(c, 0, mask, 200) == (True, False)


def test_module_is_exported_where_the_modules_are():
    assert TL.int4_route is int4_route


@pytest.mark.parametrize("name", ["layers", "batch", "max_tokens", "page_size"])
def test_sizes_of_nothing_are_refused(name):
    with pytest.raises(ValueError, match="at least 1"):
        make(**{name: 0})
