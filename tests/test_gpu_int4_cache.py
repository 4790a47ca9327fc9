"""The 4-bit cache in the models: the modules' attention over it against the 64-bit definition on
what the cache holds, whole models against the same model that reads the cache back for its own
attention, generation, cropping."""
from __future__ import annotations

import copy

import numpy as np
import pytest
import torch
from transformers import LlamaConfig, LlamaForCausalLM, Qwen2Config, Qwen2ForCausalLM

from _paged_int4 import rounded, tolerance
from oracle import paged_int4_oracle as P
from tilemix_amd.models import tilemix_llama as TL
from tilemix_amd.models import tilemix_qwen as TQ
from tilemix_amd.models.int4_cache import Int4KVCache

pytestmark = pytest.mark.gpu


def llama(heads=4, kv_heads=2, hidden=256):
    cfg = LlamaConfig(vocab_size=512, hidden_size=hidden, intermediate_size=512, num_hidden_layers=2,
                      num_attention_heads=heads, num_key_value_heads=kv_heads, rope_theta=500000.0)
    torch.manual_seed(0)
    model = LlamaForCausalLM(cfg).half().cuda().eval()
    TL.inject_tilemix_into_llama(model)
    TL.configure_tilemix_attention_pattern(model, "sptrans", percentage=0.5, stride=128, c=32)
    return model


def qwen():
    cfg = Qwen2Config(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, rope_theta=500000.0)
    torch.manual_seed(0)
    model = Qwen2ForCausalLM(cfg).half().cuda().eval()
    TQ.inject_tilemix_into_qwen(model)
    TQ.configure_tilemix_attention_pattern(model, "sptrans", percentage=0.5, stride=128, c=32)
    return model


def ids(batch, tokens, seed=1):
    return torch.randint(0, 512, (batch, tokens), generator=torch.Generator().manual_seed(seed)).cuda()


STEPS = (100, 40, 5, 1, 1, 17, 1)  # a prefill, chunks and decode steps


@pytest.mark.parametrize("dim,batch", [(64, 2), (32, 1), (128, 3)])
def test_attention_over_the_cache(monkeypatch, dim, batch):
    """Every attend call of a run, against the definition on the pools at that time; what was stored
    is the quantised K and V."""
    model = llama(heads=4, kv_heads=2, hidden=4 * dim)
    cache = Int4KVCache.for_model(model, batch, 200, page_size=32, unpadded=True)
    calls, stored = [], {0: [], 1: []}
    attend, append = Int4KVCache.attend, Int4KVCache.append

    def spy_attend(self, q, idx, scale):
        out = attend(self, q, idx, scale)
        pool = [a.cpu().numpy() for a in self.layers[idx].pool._args[:4]]
        calls.append((q.double().cpu().numpy(), idx, scale, out.double().cpu().numpy(), pool, self.layers[idx].seen))
        return out

    def spy_append(self, k, v, idx):
        append(self, k, v, idx)
        stored[idx].append((k.double().cpu().numpy(), v.double().cpu().numpy()))

    monkeypatch.setattr(Int4KVCache, "attend", spy_attend)
    monkeypatch.setattr(Int4KVCache, "append", spy_append)
    tokens = ids(batch, sum(STEPS))
    at = 0
    with torch.no_grad():
        for n in STEPS:
            assert torch.isfinite(model(tokens[:, at:at + n], past_key_values=cache).logits).all()
            at += n
            assert cache.get_seq_length() == at == int(cache.tables.seq_lens[0])
    assert len(calls) == 2 * (len(STEPS) - 1)
    table = cache.tables.block_table.cpu().numpy()
    for q, idx, scale, out, pool, seen in calls:
        b, h, t, d = q.shape
        assert out.shape == (b, t, h, d)
        cu = np.arange(0, (b + 1) * t, t)
        ref, mag, size = P.attention(q.transpose(0, 2, 1, 3).reshape(b * t, h, d), *pool, d, table, [seen] * b, cu, t, seen,
                                     True, scale)
        assert (np.abs(out.reshape(b * t, h, d) - ref) <= tolerance(ref, mag, size, d, "fp16")).all()
    for idx in (0, 1):
        for j, (codes, params) in enumerate(((0, 1), (2, 3))):
            pool = [a.cpu().numpy() for a in cache.layers[idx].pool._args[:4]]
            x = np.concatenate([s[j] for s in stored[idx]], axis=2)  # [B, H, T, D]
            want = P.dequantise(*P.quantise(x), dim)
            for b in range(batch):
                got, there = P.read_rows(pool[codes], pool[params], dim, table[b], at, pool[0].shape[0], 32)
                assert there.all() and np.array_equal(got, want[b])


@pytest.mark.parametrize("make", [llama, qwen])
def test_models_match_their_own_attention_over_the_same_cache(make):
    """unpadded: attention over the codes; else, with the eager attention's mask, the model's own attention over
    what update reads back."""
    model = make()
    eager = copy.deepcopy(model)
    eager.config._attn_implementation = "eager"
    caches = [Int4KVCache.for_model(model, 2, 200, unpadded=True), Int4KVCache.for_model(model, 2, 200)]
    tokens = ids(2, sum(STEPS), seed=3)
    at, agree, total = 0, 0, 0
    with torch.no_grad():
        for n in STEPS:
            got, ref = (m(tokens[:, at:at + n], past_key_values=c).logits.float() for m, c in zip((model, eager), caches))
            at += n
            diff = (got - ref).abs()
            assert torch.isfinite(got).all() and diff.max() < 0.05 and diff.mean() < 2e-3, (n, diff.max(), diff.mean())
            agree, total = agree + (got.argmax(-1) == ref.argmax(-1)).sum().item(), total + got.shape[0] * n
    assert agree >= 0.99 * total, (agree, total)


def test_update_reads_the_cache_back():
    """The contract of transformers' caches: the first call's tensors, then all tokens'."""
    cache = Int4KVCache(1, 2, 80, 2, 60, page_size=16)
    gen = torch.Generator().manual_seed(0)
    parts = [[torch.randn(2, 2, n, 80, generator=gen).to(torch.bfloat16).cuda() for _ in range(2)] for n in (20, 3, 1)]
    k, v = cache.update(*parts[0], 0)
    assert k is parts[0][0] and v is parts[0][1]
    for n, part in zip((23, 24), parts[1:]):
        k, v = cache.update(*part, 0)
        assert k.shape == (2, 2, n, 80) and k.dtype == torch.bfloat16
    for got, j in ((k, 0), (v, 1)):
        x = torch.cat([p[j] for p in parts], dim=2).double().cpu().numpy()
        assert np.array_equal(got.double().cpu().numpy(), rounded(P.dequantise(*P.quantise(x), 80), "bf16"))


def test_masked_calls_take_the_models_own_attention(monkeypatch):
    """A cache that was not promised unpadded sequences: with a mask nothing attends over the codes."""
    model = llama()
    cache = Int4KVCache.for_model(model, 2, 100)
    monkeypatch.setattr(Int4KVCache, "attend", lambda *a: pytest.fail("attended over the codes"))
    mask = torch.ones(2, 60, dtype=torch.long, device="cuda")
    mask[0, :7] = 0  # padded on the left
    tokens = ids(2, 60)
    with torch.no_grad():
        model(tokens[:, :40], attention_mask=mask[:, :40], past_key_values=cache)
        for at in (40, 50):
            out = model(tokens[:, at:at + 10], attention_mask=mask[:, :at + 10], past_key_values=cache)
            assert torch.isfinite(out.logits).all()
    assert cache.get_seq_length() == 60


def test_generate_crop_and_reset():
    model = llama()
    prompt = ids(2, 50, seed=5)
    cache = Int4KVCache.for_model(model, 2, 100, unpadded=True)
    with torch.no_grad():
        text = model.generate(prompt, past_key_values=cache, max_new_tokens=12, do_sample=False, eos_token_id=None,
                              pad_token_id=0)
        own = Int4KVCache.for_model(model, 2, 100, unpadded=True)
        logits = model(prompt, past_key_values=own).logits[:, -1]
        for step in range(12):
            token = logits.argmax(-1)
            assert torch.equal(token, text[:, 50 + step])
            last = logits
            logits = model(token[:, None], past_key_values=own).logits[:, -1]
        free = int(own.tables.free_count)
        # the last step once more
        own.crop(-1)
        assert own.get_seq_length() == 61 and int(own.tables.seq_lens[1]) == 61
        again = model(text[:, 61:62], past_key_values=own).logits[:, -1]
        assert torch.equal(again, logits) and int(own.tables.free_count) == free
        own.crop(-20)
        assert own.get_seq_length() == 42 and (own.tables.block_table[:, 1:] == -1).all()
        own.reset()
        assert own.get_seq_length() == 0 and int(own.tables.free_count) == own.layers[0].pool.pages
        first = model(prompt, past_key_values=own).logits[:, -1]
        assert torch.equal(first.argmax(-1), text[:, 50])


def test_a_capture_is_refused():
    """The cache counts on the host; after the refusal it goes on as if the call had not been."""
    cache = Int4KVCache(1, 2, 64, 2, 64, page_size=16)
    k = torch.randn(2, 2, 3, 64, device="cuda", dtype=torch.float16)
    cache.append(k, k, 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="no part in a graph capture"):
            cache.append(k, k, 0)
    assert cache.length == 3
    cache.append(k, k, 0)
    assert cache.length == 6 and cache.tables.seq_lens.tolist() == [6, 6]
