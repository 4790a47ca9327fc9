"""The paged 4-bit KV cache on the GPU against its 64-bit definition (oracle/paged_int4_oracle.py)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _paged_int4 import TYPES, make_pool, make_table, rounded, tolerance
from oracle import paged_int4_oracle as P
from tilemix_amd.attention.hip.paged_int4 import (PagedInt4Cache, PageTables, load_int4, paged_int4_attention,
                                                  store_int4)

pytestmark = pytest.mark.gpu


def dev(a, dtype=None):
    t = torch.from_numpy(np.array(a, order="C"))
    return (t if dtype is None else t.to(dtype)).cuda()


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def to_cache(pool, dim):
    return PagedInt4Cache(*(dev(a) for a in pool), dim)


class Call:
    """One attention call: inputs on both sides, the 64-bit result and its tolerance."""

    def __init__(self, lens, new, heads, kv_heads, dim, page=16, dtype="fp16", causal=True, scale=None, seed=0,
                 max_k=None, max_q=None):
        self.table, pages = make_table(lens, page, seed)
        self.pool = make_pool(pages, kv_heads, dim, page, seed)
        self.lens, self.new, self.dim, self.dtype, self.causal = lens, new, dim, dtype, causal
        self.cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int64)
        q = np.random.default_rng(seed + 7).standard_normal((int(self.cu[-1]), heads, dim))
        q[..., 7 % dim] *= 8.0
        self.q = rounded(q, dtype)
        self.scale = dim ** -0.5 if scale is None else scale
        self.given_scale = scale
        self.max_q = max(new, default=0) if max_q is None else max_q
        self.max_k = max(lens, default=0) if max_k is None else max_k

    def want(self):
        ref, mag, size = P.attention(self.q, *self.pool, self.dim, self.table, self.lens, self.cu, self.max_q,
                                     self.max_k, self.causal, self.scale)
        return ref, tolerance(ref, mag, size, self.dim, self.dtype)

    def device_args(self):
        return (dev(self.q, TYPES[self.dtype]), to_cache(self.pool, self.dim), dev(self.table), ints(self.lens),
                dev(self.cu, torch.int32), self.max_q, self.max_k)

    def run(self, **kw):
        return paged_int4_attention(*self.device_args(), causal=self.causal, sm_scale=self.given_scale, **kw)

    def check(self, got=None):
        got = self.run() if got is None else got
        ref, tol = self.want()
        assert got.dtype == TYPES[self.dtype] and got.shape == ref.shape
        diff = np.abs(got.double().cpu().numpy() - ref)
        assert np.isfinite(diff).all() and (diff <= tol).all(), f"worst {np.max(diff / tol):.2f} of the tolerance"


def want_on_gpu(c):
    """Call.want for large calls: the same formulas in float64 on the GPU."""
    def values(codes, params):
        codes, params = dev(codes), dev(params).double()
        n = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).double()
        s, m = (params[..., i].repeat_interleave(P.GROUP, dim=-1) for i in (0, 1))
        return (n * s + m).half().double()[..., :c.dim]

    kp, vp = values(*c.pool[:2]), values(*c.pool[2:])
    pages, hk, page = kp.shape[:3]
    q = dev(c.q)
    out, mag, size = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64).cuda()
    for b, n in enumerate(c.lens):
        rows = slice(int(c.cu[b]), int(c.cu[b + 1]))
        nq = rows.stop - rows.start
        if n == 0 or nq == 0:
            continue
        ids = dev(c.table[b, :-(-n // page)]).long()
        ok = (ids >= 0) & (ids < pages)
        safe = ids.clamp(0, pages - 1)
        there = ok.repeat_interleave(page)[:n]
        limit = torch.arange(n - nq, n).cuda() if c.causal else torch.full((nq,), n - 1).cuda()
        seen = there[None, :] & (torch.arange(n).cuda()[None, :] <= limit[:, None])
        for h in range(q.shape[1]):
            k, v = (x[safe, h // (q.shape[1] // hk)].reshape(-1, c.dim)[:n] * there[:, None] for x in (kp, vp))
            s = (q[rows, h] @ k.T * c.scale).masked_fill(~seen, float("-inf"))
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(top.isinf(), 0.0, top))
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            out[rows, h], mag[rows, h] = p @ v, p @ v.abs()
            size[rows, h] = (q[rows, h].abs() @ k.abs().T * abs(c.scale)).masked_fill(~seen, 0.0).amax(-1)
    ref, mag, size = (x.cpu().numpy() for x in (out, mag, size))
    return ref, tolerance(ref, mag, size, c.dim, c.dtype)


# ---- page tables -------------------------------------------------------------------


def host_tables(tables):
    return (tables.block_table.tolist(), tables.seq_lens.tolist(), tables.free_pages.tolist(),
            int(tables.free_count))


@pytest.mark.parametrize("batch,page,pages,steps", [(1, 16, 4, 12), (3, 16, 9, 30), (65, 64, 300, 8), (300, 32, 999, 6),
                                                    (513, 16, 100, 5), (4096, 16, 3000, 3)])
def test_tables_follow_the_definition(batch, page, pages, steps):
    """Random extensions (too long, negative and empty ones among them; too few pages) and cuts."""
    rng = np.random.default_rng(batch)
    columns = 7
    tables = PageTables.empty(pages, batch, columns, page)
    table, lens, stack, count = host_tables(tables)
    for step in range(steps):
        new = [int(x) for x in rng.choice([0, 1, 1, 2, page - 1, page, page + 1, 3 * page, 8 * page, -1], batch)]
        tokens = max(0, sum(max(n, 0) for n in new) - int(rng.integers(0, 3) == 0) * page)
        slots, positions, cu, granted, count = P.extend(table, lens, stack, count, new, page, tokens)
        plan = tables.extend(ints(new), tokens)
        assert plan.slots.tolist() == slots and plan.positions.tolist() == positions
        assert plan.cu_seqlens.tolist() == cu and plan.granted.tolist() == granted
        assert plan.slots.dtype == plan.positions.dtype == torch.int64
        assert host_tables(tables)[0] == table and host_tables(tables)[1] == lens
        assert int(tables.free_count) == count and tables.free_pages.tolist()[:count] == stack[:count]
        keep = [int(x) for x in rng.choice([0, -5, 1, page, 10 * page, 10 * page, 10 * page], batch)]
        count = P.truncate(table, lens, stack, count, keep, page)
        tables.truncate(ints(keep))
        assert host_tables(tables)[:2] == (table, lens)
        assert int(tables.free_count) == count and tables.free_pages.tolist()[:count] == stack[:count]
    used = [p for row in table for p in row if p >= 0]
    assert sorted(used + stack[:count]) == list(range(pages))


def test_tables_cut_undoes_an_extension():
    tables = PageTables.empty(500, 40, 20, 16)
    rng = np.random.default_rng(0)
    tables.extend(ints(rng.integers(0, 90, 40).tolist()), 4000)
    before = [t.clone() for t in (tables.block_table, tables.seq_lens, tables.free_pages, tables.free_count)]
    tables.extend(ints(rng.integers(0, 70, 40).tolist()), 4000)
    tables.truncate(before[1])
    for a, b in zip(before, (tables.block_table, tables.seq_lens, tables.free_pages, tables.free_count)):
        assert torch.equal(a, b)


def test_tables_of_no_sequence_and_no_token():
    tables = PageTables.empty(4, 0, 3, 16)
    plan = tables.extend(ints([]), 0)
    assert plan.cu_seqlens.tolist() == [0] and plan.granted.numel() == plan.slots.numel() == 0
    tables.truncate(ints([]))
    tables = PageTables.empty(4, 2, 3, 16)
    plan = tables.extend(ints([0, 0]), 0)
    assert plan.cu_seqlens.tolist() == [0, 0, 0] and plan.granted.tolist() == [1, 1]
    plan = tables.extend(ints([0, 3]), 9)  # entries that no sequence needs
    assert plan.slots.tolist() == [0, 1, 2] + [-1] * 6 and plan.positions.tolist() == [0, 1, 2] + [0] * 6


def test_tables_with_state_out_of_range():
    """Lengths, counts and pages that no call leaves behind stay within the arrays."""
    tables = PageTables.empty(4, 3, 2, 16)
    tables.seq_lens.copy_(ints([-7, 10 ** 9, 5]))
    tables.free_count.fill_(1000)
    tables.free_pages.copy_(ints([3, -9, 2 ** 31 - 1, 0]))
    plan = tables.extend(ints([20, 2 ** 31 - 1, 1]), 64)
    assert plan.granted.tolist() == [1, 0, 0]  # the second request's end is past num_tokens, and so is the third's
    assert tables.block_table[0].tolist() == [0, 2 ** 31 - 1] and tables.seq_lens.tolist() == [20, 32, 5]
    tables.truncate(ints([-3, 0, 0]))
    assert tables.seq_lens.tolist() == [0, 0, 0] and int(tables.free_count) == 4


# ---- rows ---------------------------------------------------------------------------


@pytest.mark.parametrize("dim,heads,page,dtype", [(128, 8, 64, "fp16"), (128, 1, 16, "bf16"), (96, 2, 32, "fp16"),
                                                  (80, 3, 16, "bf16"), (64, 2, 48, "fp16"), (33, 2, 16, "fp16"),
                                                  (32, 1, 16, "bf16"), (7, 2, 16, "fp16"), (1, 1, 16, "fp16")])
def test_store_and_load(dim, heads, page, dtype):
    """Stored rows are the definition's codes and parameters, bit for bit, others stay, and load
    returns the values they stand for."""
    lens = [1, 0, page, page + 1, 3 * page - 1, 37]
    table, pages = make_table(lens, page, dim)
    pool = make_pool(pages, heads, dim, page, dim)
    before = [a.copy() for a in pool]
    cache = to_cache(pool, dim)
    rng = np.random.default_rng(dim)
    slots = [int(table[b, t // page]) * page + t % page for b, n in enumerate(lens) for t in range(n)]
    skipped = [-1, pages * page, -2 ** 40, 2 ** 40]
    order = rng.permutation(len(slots) + len(skipped))
    where = np.array(slots + skipped, dtype=np.int64)[order]
    x = {}
    for name in "kv":
        v = rng.standard_normal((len(where), heads, dim)) * rng.choice([1e-3, 1.0, 300.0], (len(where), heads, 1))
        v[0] = 0.0
        v[1] = 5.0
        v[2, :, 0] = 6e4
        v[3, :, -1] = -6e4
        x[name] = rounded(v, dtype)
    store_int4(dev(x["k"], TYPES[dtype]), dev(x["v"], TYPES[dtype]), cache, dev(where))
    for name, at in (("k", 0), ("v", 2)):
        codes, params = P.quantise(x[name])
        for t, slot in enumerate(where):
            if 0 <= slot < pages * page:
                before[at][slot // page, :, slot % page] = codes[t]
                before[at + 1][slot // page, :, slot % page] = params[t]
    for a, b in zip(before, (cache.k_codes, cache.k_params, cache.v_codes, cache.v_params)):
        assert np.array_equal(a.view(np.uint8), b.cpu().numpy().view(np.uint8))
    cu = np.concatenate([[0], np.cumsum(lens)])
    for out_type in TYPES:
        k, v = load_int4(cache, dev(table), ints(cu.tolist()), int(cu[-1]) + 5, dtype=TYPES[out_type])
        for got, at in ((k, 0), (v, 2)):
            want = np.zeros((int(cu[-1]) + 5, heads, dim))
            for b, n in enumerate(lens):
                want[cu[b]:cu[b + 1]] = P.read_rows(before[at], before[at + 1], dim, table[b], n, pages,
                                                    page)[0].transpose(1, 0, 2)
            assert got.dtype == TYPES[out_type]
            assert np.array_equal(got.double().cpu().numpy(), rounded(want, out_type))


def test_store_of_strided_and_special_rows():
    """Head-major and sliced K and V; infinities and finite values past the limit are clamped, a NaN
    makes its group NaN and no other."""
    dim, heads, page = 128, 2, 16
    pool = make_pool(3, heads, dim, page)
    rng = np.random.default_rng(3)
    big = rng.standard_normal((heads, 9, 2 * dim + 3))
    big[0, 0, 5], big[1, 2, 40], big[0, 3, 70], big[1, 4, 3] = np.inf, -np.inf, np.nan, 65504.0
    t = torch.from_numpy(big).half().cuda()
    for k in (t.transpose(0, 1)[..., :dim], t.transpose(0, 1)[..., 3:dim + 3], t.transpose(0, 1)[..., 0:2 * dim:2]):
        cache = to_cache(pool, dim)
        store_int4(k, k.contiguous(), cache, torch.arange(4, 13).cuda())
        codes, params = P.quantise(k.double().cpu().numpy())
        for c, p in ((cache.k_codes, cache.k_params), (cache.v_codes, cache.v_params)):
            got_c = torch.cat([c[0, :, 4:16], c[1, :, :0]], 1)[:, :9].transpose(0, 1).cpu().numpy()
            got_p = p[0, :, 4:13].transpose(0, 1).cpu().numpy()
            assert np.array_equal(got_c, codes)
            assert np.array_equal(np.isnan(got_p), np.isnan(params))
            assert np.array_equal(np.nan_to_num(got_p), np.nan_to_num(params))
            assert np.isfinite(P.dequantise(got_c, got_p, dim)[~np.isnan(params).any((-1, -2))]).all()


def test_store_rounding_of_every_quotient():
    """Rows of fp16 neighbours of the code borders: the codes are those of an exact division."""
    rng = np.random.default_rng(5)
    dim, page, tokens = 128, 16, 512
    low = rng.uniform(-4, 0, (tokens, 1, 4, 1))
    span = np.float16(rng.uniform(0.01, 8, (tokens, 1, 4, 1))).astype(np.float64)
    step = (span / 15).astype(np.float16).astype(np.float64)
    x = low + (rng.integers(0, 15, (tokens, 1, 4, 32)) + 0.5) * step
    x[..., 0], x[..., 1] = low[..., 0], (low + span)[..., 0]
    x = rounded(x.reshape(tokens, 1, dim), "fp16")
    cache = PagedInt4Cache.empty(tokens // page, 1, dim, page)
    t = dev(x, torch.float16)
    store_int4(t, t, cache, torch.arange(tokens).cuda())
    codes, params = P.quantise(x)
    assert np.array_equal(cache.k_codes.reshape(tokens, 1, -1).cpu().numpy(), codes)
    assert np.array_equal(cache.v_params.reshape(tokens, 1, 4, 2).cpu().numpy(), params)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_store_ties_and_odd_groups_side_by_side(dtype):
    """Exact halves between two codes go to the even one; ranges below fp16's normal numbers, constant groups, values
    beyond the limit, infinities and NaN take their own way within a wave, in any company."""
    rng = np.random.default_rng(11)
    dim, page, tokens = 128, 16, 640
    x = np.zeros((tokens, 2, 4, 32))
    kind = rng.integers(0, 9, (tokens, 2, 4))
    kind[:64], kind[64:128] = 0, 1  # (whole waves of ties)
    for at in np.ndindex(*kind.shape):
        n, k = rng.integers(0, 16, 32), kind[at]
        n[:2] = 0, 15
        if k in (0, 1):  # minimum, then halves: quotients k + 1/2 exactly
            step = 2.0 ** rng.integers(-6, 3)
            x[at] = (n + np.where((n < 15) & (n > 0), 0.5, 0.0)) * step - 8 * step * k
        elif k == 2:  # a range of a few of fp16's smallest steps
            x[at] = rng.integers(-9, 25, 32) * 2.0 ** -24
        elif k == 3:
            x[at] = rng.standard_normal()
        elif k == 4:  # a minimum that fp16 does not have, a narrow range
            x[at] = 1000.0 + rng.uniform(0, 8, 32)
        elif k == 5:
            x[at] = rng.choice([65408.0, 65472.0, 65504.0, -65504.0, 3.0], 32)
        elif k == 6:
            x[at] = np.where(rng.random(32) < 0.1, rng.choice([np.inf, -np.inf], 32), rng.standard_normal(32))
        elif k == 7:
            x[at] = np.where(rng.random(32) < 0.1, np.nan, rng.standard_normal(32))
        else:
            x[at] = rng.standard_normal(32)
    x = rounded(x.reshape(tokens, 2, dim), dtype)
    cache = PagedInt4Cache.empty(tokens // page, 2, dim, page)
    t = dev(x, TYPES[dtype])
    store_int4(t, t.flip(0), cache, torch.arange(tokens).cuda())
    codes, params = P.quantise(x)
    for got, want in ((cache.k_codes, codes), (cache.v_codes, codes[::-1])):
        assert np.array_equal(got.transpose(1, 2).reshape(tokens, 2, -1).cpu().numpy(), want)
    for got, want in ((cache.k_params, params), (cache.v_params, params[::-1])):
        got = got.transpose(1, 2).reshape(tokens, 2, 4, 2).cpu().numpy()
        assert np.array_equal(got, want.reshape(got.shape), equal_nan=True)


def test_load_of_pages_that_are_not_there():
    """Table entries out of range and tokens past the table's columns read as zeros."""
    dim, page = 64, 16
    pool = make_pool(4, 2, dim, page)
    table = np.array([[2, -1, 4, 1], [2 ** 31 - 1, 0, -2 ** 31, 3]], dtype=np.int32)
    cu = [0, 70, 130]
    k, v = load_int4(to_cache(pool, dim), dev(table), ints(cu), 130)
    for got, at in ((k, 0), (v, 2)):
        want = np.concatenate([P.read_rows(pool[at], pool[at + 1], dim, table[b], cu[b + 1] - cu[b], 4,
                                           page)[0].transpose(1, 0, 2) for b in range(2)])
        assert np.array_equal(got.double().cpu().numpy(), want)
    assert not v[64:70].any()


# ---- attention ----------------------------------------------------------------------


@pytest.mark.parametrize("lens", [[1], [2, 0, 1], [15, 16, 17], [63, 64, 65], [127, 129, 255, 256, 257, 300]])
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 6, 2), (64, 7, 1)])
def test_decode(lens, dim, heads, kv_heads):
    Call(lens, [1] * len(lens), heads, kv_heads, dim).check()


@pytest.mark.parametrize("dim", [1, 8, 16, 31, 32, 40, 64, 72, 80, 96, 100, 112, 128])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_head_dims(dim, dtype):
    Call([100, 37], [1, 3], 4, 2, dim, dtype=dtype, seed=dim).check()


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (14, 2), (28, 4), (16, 1), (17, 1), (40, 2), (33, 1),
                                            (130, 1)])
def test_grouped_heads(heads, kv_heads):
    """Up to, at and past the 16 and 32 rows of a block with a single query."""
    Call([70, 5], [1, 1], heads, kv_heads, 64, seed=heads).check()


@pytest.mark.parametrize("page", [16, 32, 48, 64, 128, 208])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_page_sizes(page, dtype):
    """Pages that end inside a tile, whole tiles and more than one; 48 and 208 divide none."""
    Call([500, 63, 1, 209], [1, 2, 1, 5], 6, 2, 128, page=page, dtype=dtype, seed=page).check()


@pytest.mark.parametrize("new", [[2, 2, 2], [5, 1, 16], [17, 30, 70], [0, 64, 1], [70, 0, 33], [90, 200, 1]])
@pytest.mark.parametrize("causal", [True, False])
def test_several_queries(new, causal):
    """Drafts and chunks; more queries than keys leave the first rows without any."""
    Call([90, 200, 33], new, 6, 2, 128, causal=causal, seed=sum(new)).check()


@pytest.mark.parametrize("new", [[300], [129, 1]])
@pytest.mark.parametrize("dim,heads,kv_heads,dtype", [(128, 3, 1, "fp16"), (64, 4, 2, "bf16"), (96, 2, 1, "fp16"),
                                                      (40, 5, 1, "bf16")])
def test_chunks(new, dim, heads, kv_heads, dtype):
    Call([700, 140][:len(new)], new, heads, kv_heads, dim, page=64, dtype=dtype, seed=dim).check()


@pytest.mark.parametrize("lens,new,heads,kv_heads,dim", [([5000], [1], 4, 2, 64), ([9000, 33, 2100], [1, 1, 1], 2, 1, 128),
                                                         ([6001], [4], 6, 1, 96), ([4097, 700], [40, 3], 2, 1, 32)])
def test_long_sequences_are_split(lens, new, heads, kv_heads, dim):
    Call(lens, new, heads, kv_heads, dim, page=64, seed=dim).check()


CHUNKS = {  # more than 96 rows a (sequence, KV head) and 10000 tiles of 32 rows: operands shared by the workgroup
    "one": dict(lens=[6003], new=[1200], heads=3, kv_heads=1, dim=128, page=64),
    "ragged": dict(lens=[5000, 33, 1207, 64, 0, 700], new=[700, 33, 5, 1, 0, 699], heads=6, kv_heads=2, dim=128, page=32),
    "d64_bf16": dict(lens=[3001, 3000], new=[500, 1], heads=14, kv_heads=2, dim=64, page=16, dtype="bf16"),
    "d96": dict(lens=[2900, 100], new=[900, 100], heads=8, kv_heads=2, dim=96, page=48),
    "d40": dict(lens=[6000], new=[999], heads=8, kv_heads=2, dim=40, page=128, dtype="bf16"),
    "d32": dict(lens=[4100, 64], new=[600, 200], heads=8, kv_heads=2, dim=32, page=16),
    "all_see": dict(lens=[2500, 65], new=[1000, 3], heads=4, kv_heads=2, dim=128, page=64, causal=False),
    "more_queries_than_keys": dict(lens=[1500, 900], new=[2000, 901], heads=4, kv_heads=2, dim=128, page=64),
    "split": dict(lens=[70000, 60000], new=[45, 33], heads=3, kv_heads=1, dim=128, page=64),
    "split_bf16_d64": dict(lens=[70001], new=[60], heads=7, kv_heads=1, dim=64, page=64, dtype="bf16"),
}


@pytest.mark.parametrize("name", CHUNKS)
def test_chunk_kernel(name):
    c = Call(seed=len(name), **CHUNKS[name])
    hk, rows = c.pool[0].shape[1], c.max_q * c.q.shape[1] // c.pool[0].shape[1]
    assert rows > 96 and -(-rows // 32) * hk * len(c.lens) * -(-c.max_k // 64) > 10000
    got = c.run()
    ref, tol = want_on_gpu(c)
    diff = np.abs(got.double().cpu().numpy() - ref)
    assert np.isfinite(diff).all() and (diff <= tol).all(), f"worst {np.max(diff / tol):.2f} of the tolerance"


def lengths(n, high, seed, low=0):
    return [int(x) for x in np.random.default_rng(seed).integers(low, high + 1, n)]


RAGGED = {  # batches whose keys are shared out by the sequences' lengths, more than 64 of them among those
    "decode": dict(lens=lengths(150, 2500, 1), new=[1] * 150, heads=4, kv_heads=2, dim=64, page=32),
    "decode_with_idle": dict(lens=lengths(70, 3000, 2), new=lengths(70, 1, 3), heads=3, kv_heads=3, dim=128, page=64),
    "one_long": dict(lens=[30000] + lengths(9, 90, 4), new=[1] * 10, heads=6, kv_heads=2, dim=96, page=16, dtype="bf16"),
    "nothing_but_one": dict(lens=[0] * 40 + [5000] + [0] * 40, new=[1] * 81, heads=2, kv_heads=1, dim=64, page=64),
    "drafts": dict(lens=lengths(66, 2400, 5), new=lengths(66, 9, 6), heads=8, kv_heads=2, dim=64, page=16),
    "drafts_few": dict(lens=[6100, 17, 0, 1500, 3300], new=[6, 6, 0, 6, 1], heads=24, kv_heads=8, dim=128, page=64),
    "drafts_33": dict(lens=lengths(20, 4000, 7, 33), new=[33] * 20, heads=4, kv_heads=4, dim=32, page=48),
    "see_all": dict(lens=lengths(12, 4000, 8), new=lengths(12, 12, 9), heads=8, kv_heads=4, dim=128, page=64, causal=False),
    "chunks": dict(lens=lengths(70, 2900, 10, 300), new=[300] + lengths(69, 3, 11), heads=2, kv_heads=1, dim=64, page=64),
    "chunks_few": dict(lens=[9000, 300, 4000], new=[200, 300, 50], heads=24, kv_heads=8, dim=128, page=64),
}


@pytest.mark.parametrize("name", RAGGED)
def test_ragged_batches(name):
    c = Call(seed=len(name), **RAGGED[name])
    got = c.run()
    ref, tol = want_on_gpu(c)
    diff = np.abs(got.double().cpu().numpy() - ref)
    assert np.isfinite(diff).all() and (diff <= tol).all(), f"worst {np.max(diff / tol):.2f} of the tolerance"
    assert torch.equal(c.run(), got)


def test_ragged_batch_in_a_graph_follows_the_lengths():
    """Lengths that change between the replays: the pieces are found anew."""
    c = Call(lengths(40, 3000, 12, 1), [1] * 40, 4, 2, 64, page=32, seed=12)
    q, cache, table, lens, cu, max_q, max_k = c.device_args()
    run = lambda: paged_int4_attention(q, cache, table, lens, cu, max_q, max_k)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in range(4):
        c.lens = [min(a, b) for a, b in zip(c.lens, lengths(40, 3000 >> seed, 20 + seed, 1))]
        lens.copy_(ints(c.lens))
        graph.replay()
        torch.cuda.synchronize()
        c.check(out)
        assert torch.equal(run(), out)


@pytest.mark.parametrize("new,heads", [(1, 4), (6, 8), (300, 2)])
def test_queries_out_of_order_stay_inside(new, heads):
    """Starts of sequences that do not ascend: nobody else's memory is touched, and the next call is right."""
    lens = lengths(40, 2900, 13, 1500)
    c = Call(lens, [new] * 40, heads, 1, 64, page=64, seed=13)
    q, cache, table, seq, cu, max_q, max_k = c.device_args()
    room = torch.full((q.shape[0] + 8, heads, 64), 9.0, dtype=torch.float16, device="cuda")
    for bad in (cu.flip(0), torch.where(torch.arange(41, device="cuda") % 2 == 0, cu * 0, cu), cu * 0 - 5, cu * 0 + 2 ** 30):
        paged_int4_attention(q, cache, table, seq, bad.int().contiguous(), max_q, max_k, out=room[4:-4])
        assert (room[:4] == 9.0).all() and (room[-4:] == 9.0).all()
    got = c.run()
    ref, tol = want_on_gpu(c)
    assert (np.abs(got.double().cpu().numpy() - ref) <= tol).all()


def test_chunk_kernel_pages_nan_and_what_lies_behind():
    """Bad pages, stale rows behind the end and a stored NaN, with operands shared by the workgroup."""
    c = Call([3000, 700], [1000, 40], 6, 2, 128, page=16, seed=21)
    ref, tol = want_on_gpu(c)
    clean = c.run().double().cpu().numpy()
    assert (np.abs(clean - ref) <= tol).all()
    used = np.zeros(c.pool[0].shape[0] * 16, dtype=bool)
    for b, n in enumerate(c.lens):
        for t in range(n):
            used[int(c.table[b, t // 16]) * 16 + t % 16] = True
    used = used.reshape(-1, 16)
    for at in (1, 3):
        c.pool[at][~used.repeat(2, axis=0).reshape(-1, 2, 16)] = np.nan
    assert np.array_equal(c.run().double().cpu().numpy(), clean)
    # V of KV head 1, group 1, key 2500 of sequence 0: queries from 500 on see it
    c.pool[3][c.table[0, 2500 // 16], 1, 2500 % 16, 1, 0] = np.nan
    got = c.run().double().cpu().numpy()
    want = clean.copy()
    want[500:1000, 3:, 32:64] = np.nan
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~np.isnan(want)], clean[~np.isnan(want)])
    c = Call([3000, 700], [1000, 40], 6, 2, 128, page=16, seed=21)
    c.table[0, 3], c.table[0, 100], c.table[0, 187] = -1, 10 ** 9, -2 ** 31
    c.table[1, :] = -7
    ref, tol = want_on_gpu(c)
    got = c.run().double().cpu().numpy()
    assert (np.abs(got - ref) <= tol).all() and not got[1000:].any()


def test_chunk_kernel_out_and_graph():
    """Strided q and out, rows behind the last query, one captured call replayed on changed inputs."""
    c = Call([2600, 100], [900, 3], 6, 2, 128, page=64, seed=22)
    q, *rest = c.device_args()
    clean = paged_int4_attention(q, *rest)
    wide = torch.zeros(910, 6, 133, dtype=torch.float16, device="cuda")
    wide[:903, :, 3:131] = q
    out = torch.full((6, 910, 140), 9.0, dtype=torch.float16, device="cuda").transpose(0, 1)
    paged_int4_attention(wide[:, :, 3:131], *rest, out=out[:, :, 5:133])
    assert torch.equal(out[:903, :, 5:133], clean)
    assert (out[903:] == 9.0).all() and (out[:, :, :5] == 9.0).all() and (out[:, :, 133:] == 9.0).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = paged_int4_attention(q, *rest)
    lens = rest[2]
    for step in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(step)).half())
        lens.copy_(ints([2600 - 300 * step, 100 - step]))
        want = paged_int4_attention(q, *rest)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, want)


@pytest.mark.parametrize("scale", [0.0, -0.2, 0.5, 1e-30])
def test_scales(scale):
    Call([130, 20], [1, 4], 4, 2, 64, scale=scale, seed=11).check()


def test_bounds_on_queries_and_keys():
    """max_seqlen_q and max_seqlen_k cut; without cu_seqlens_q every sequence has max_seqlen_q queries."""
    Call([300, 50], [1, 1], 4, 2, 64, max_k=130).check()
    c = Call([100, 90], [3, 3], 4, 2, 64)
    q, cache, table, lens, _, max_q, max_k = c.device_args()
    c.check(paged_int4_attention(q, cache, table, lens, None, max_q, max_k))
    c = Call([100, 90], [9, 3], 4, 2, 64, max_q=5)
    args = c.device_args()
    out = torch.full_like(args[0], 7.0)
    got = paged_int4_attention(*args, out=out)
    assert (got[5:9] == 7.0).all()
    ref, tol = c.want()
    diff = np.abs(got.double().cpu().numpy() - ref)
    keep = [i for i in range(12) if not 5 <= i < 9]
    assert (diff[keep] <= tol[keep]).all()


@pytest.mark.parametrize("lens,new", [([900, 40], [3, 1]), ([6000, 2000, 2500], [40, 1, 90])])
def test_loose_bounds_cost_nothing(lens, new):
    """max_seqlen_q and max_seqlen_k far above what there is: the same values."""
    c = Call(lens, new, 6, 2, 64, page=16, seed=31, max_q=2 ** 28, max_k=2 ** 31 - 1)
    c.check()


def test_empty_calls():
    c = Call([0, 0], [1, 2], 4, 2, 64)
    assert not c.run().any()
    pool = make_pool(2, 2, 64, 16)
    q = torch.zeros(0, 4, 64, dtype=torch.float16, device="cuda")
    none = torch.empty(0, 3, dtype=torch.int32, device="cuda")
    assert paged_int4_attention(q, to_cache(pool, 64), none, ints([]), ints([0]), 1, 5).shape == q.shape
    # a table without columns: no key
    q = torch.ones(2, 4, 64, dtype=torch.float16, device="cuda")
    none = torch.empty(2, 0, dtype=torch.int32, device="cuda")
    assert not paged_int4_attention(q, to_cache(pool, 64), none, ints([5, 1]), None, 1, 5).any()


def test_out_strides_and_rows_behind():
    """q and out as slices of wider tensors, head-major, unaligned; rows behind the last query stay."""
    c = Call([90, 40], [2, 1], 4, 2, 64, seed=2)
    q, *rest = c.device_args()
    wide = torch.zeros(5, 4, 200, dtype=torch.float16, device="cuda")
    for at in (0, 3, 8):
        wide[:3, :, at:at + 64] = q
        out = torch.full((4, 5, 77), 9.0, dtype=torch.float16, device="cuda").transpose(0, 1)
        got = paged_int4_attention(wide[:, :, at:at + 64], *rest, out=out[:, :, 5:69])
        assert got.data_ptr() == out[:, :, 5:69].data_ptr()
        c.check(got[:3])
        assert (out[3:] == 9.0).all() and (out[:, :, :5] == 9.0).all() and (out[:, :, 69:] == 9.0).all()
    split = q.repeat(1, 1, 2)[:, :, ::2]  # no unit stride: copied
    assert split.stride(2) == 2
    assert torch.equal(paged_int4_attention(split, *rest), paged_int4_attention(split.contiguous(), *rest))


@pytest.mark.parametrize("lens,new,heads,kv_heads", [([90, 40], [2, 1], 4, 2), ([5000], [1], 4, 2), ([300, 290], [300, 129], 6, 2),
                                                     ([900], [70], 4, 1)])
def test_out_may_be_q(lens, new, heads, kv_heads):
    c = Call(lens, new, heads, kv_heads, 64, seed=8)
    q, *rest = c.device_args()
    want = paged_int4_attention(q, *rest)
    assert torch.equal(paged_int4_attention(q, *rest, out=q), want) and not want.isnan().any()


def test_out_may_be_q_of_a_chunk():
    c = Call(seed=3, **CHUNKS["one"])
    q, *rest = c.device_args()
    want = paged_int4_attention(q, *rest)
    assert torch.equal(paged_int4_attention(q, *rest, out=q), want) and not want.isnan().any()


def test_bad_pages_are_not_seen():
    """Table entries out of range, in the middle and for a whole sequence."""
    c = Call([200, 100, 60], [1, 2, 1], 4, 2, 64, seed=4)
    c.table[0, 1], c.table[0, 5], c.table[0, 12] = -1, 10 ** 9, -2 ** 31
    c.table[2, :] = 2 ** 31 - 1
    c.check()
    assert not c.run()[3].any()


@pytest.mark.parametrize("where", ["params", "both"])
def test_what_lies_behind_the_end_is_not_seen(where):
    """Rows behind a sequence's last token hold NaN scales and any codes."""
    c = Call([70, 16, 33], [3, 1, 20], 4, 2, 128, seed=5)
    good = c.run()
    page = 16
    bad = [a.copy() for a in c.pool]
    used = set()
    for b, n in enumerate(c.lens):
        for t in range(n):
            used.add((int(c.table[b, t // page]), t % page))
    for p in range(bad[0].shape[0]):
        for r in range(page):
            if (p, r) not in used:
                for i in (1, 3):
                    bad[i][p, :, r] = np.nan
                if where == "both":
                    bad[0][p, :, r] = bad[2][p, :, r] = 255
    c.pool = bad
    assert torch.equal(c.run(), good)


def test_nan_reaches_the_queries_that_see_it():
    """A NaN in K: all of a query's channels.  In V: the group's channels.  Earlier queries: none."""
    for at, kind in ((195, "k"), (195, "v"), (20, "v"), (199, "v")):
        c = Call([200], [16], 4, 2, 128, seed=6)
        clean = c.run().double().cpu().numpy()
        params = c.pool[1 if kind == "k" else 3]
        params[c.table[0, at // 16], 1, at % 16, 2, 1] = np.nan
        got = c.run().double().cpu().numpy()
        want = clean.copy()
        for i in range(16):
            if 200 - 16 + i >= at:
                want[i, 2:, :] = np.nan if kind == "k" else want[i, 2:, :]
                want[i, 2:, 64:96] = np.nan
        assert np.array_equal(np.isnan(got), np.isnan(want))
        seen = ~np.isnan(want)
        ref, tol = Call([200], [16], 4, 2, 128, seed=6).want()
        assert (np.abs(got - ref)[seen] <= tol[seen]).all()


def test_infinite_and_large_queries():
    """A NaN or infinite query poisons its own rows alone; bf16 queries past fp16's range work."""
    c = Call([100, 50], [4, 1], 4, 2, 64, dtype="bf16", seed=8)
    q, *rest = c.device_args()
    clean = paged_int4_attention(q, *rest)
    q[1, 2, 5] = float("nan")
    q[4, 0, 0] = float("inf")
    got = paged_int4_attention(q, *rest)
    assert got[1, 2].isnan().all() and got[4, 0].isnan().all()
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[1, 2] = hit[4, 0] = True
    assert torch.equal(got[~hit], clean[~hit])
    c = Call([60], [2], 4, 2, 64, dtype="bf16", scale=1e-7, seed=9)
    c.q = rounded(c.q * 2.0 ** 20, "bf16")
    c.check()
    c.q, c.given_scale, c.scale = rounded(c.q * 2.0 ** -60, "bf16"), 2.0 ** 40, 2.0 ** 40
    c.check()


def test_small_weights_of_many_keys_count():
    """One key 18 above 40000 others: together they weigh 0.06% (2^-26 each, below what fp16 holds beside a weight
    of one); V is 0 at the one and 1 at the others, so that the output is their share.  Held 2^7 times larger they
    are 2^-19, of fp16's steps of 2^-24: off by 2^-6 at most, beside the output's own rounding."""
    dim, page, n = 64, 64, 40001
    pages = -(-n // page)
    pool = [np.zeros((pages, 1, page, 32), np.uint8), np.zeros((pages, 1, page, 2, 2), np.float16)] * 2
    pool = [a.copy() for a in pool]
    pool[1][0, 0, 0, 0, 1] = 18.0 / 32  # K: 18 / 32 in group 0 of key 0
    pool[3][..., 1] = 1.0
    pool[3][0, 0, 0, :, 1] = 0.0
    table = np.arange(pages, dtype=np.int32)[None]
    for tokens, group in ((1, 1), (1, 20), (130, 4)):
        q = np.ones((tokens, group, dim))
        got = paged_int4_attention(dev(q, torch.float16), to_cache(pool, dim), dev(table), ints([n]), ints([0, tokens]),
                                   tokens, n, sm_scale=1.0)
        seen = n - tokens + np.arange(tokens)  # of the others
        want = (seen / (seen + np.exp(18.0)))[:, None, None]
        assert (np.abs(got.double().cpu().numpy() - want) <= (2.0 ** -6 + 2.0 ** -11) * want).all()


def test_offsets_past_32_bits():
    """A pool whose codes take more than 4 GiB: the same rows in its first and its last pages."""
    dim, heads, page = 128, 8, 64
    pages = (1 << 32) // (heads * page * 64) + 40
    cache = PagedInt4Cache.empty(pages, heads, dim, page)
    assert cache.k_codes.numel() > 1 << 32
    gen = torch.Generator().manual_seed(0)
    lens = [900, 130]
    k, v = (torch.randn(sum(lens), heads, dim, generator=gen).half().cuda() for _ in range(2))
    cu = [0, 900, 1030]
    results = []
    for new in ([1, 1], [300, 2], [900, 130]):
        q = torch.randn(sum(new), 24, dim, generator=gen).half().cuda()
        for base in (0, pages - 20):
            table = torch.full((2, 15), -1, dtype=torch.int32)
            table[0], table[1, :3] = torch.arange(base, base + 15), torch.arange(base + 15, base + 18)
            slots = torch.cat([table[b, torch.arange(n) // page].long() * page + torch.arange(n) % page
                               for b, n in enumerate(lens)])
            store_int4(k, v, cache, slots.cuda())
            out = paged_int4_attention(q, cache, table.cuda(), ints(lens), ints([0, new[0], sum(new)]), max(new), 900)
            results.append((out, *load_int4(cache, table.cuda(), ints(cu), 1030)))
    for low, high in zip(results[::2], results[1::2]):
        assert all(torch.equal(a, b) for a, b in zip(low, high))


def test_lengths_past_the_table_and_offsets_out_of_range():
    """seq_lens of more than a row's places, negative ones, cu_seqlens that start or end out of range."""
    c = Call([100, 64], [3, 2], 4, 2, 64, seed=31)
    q, cache, table, lens, cu, max_q, _ = c.device_args()
    want = paged_int4_attention(q, cache, table[:, :4], ints([64, 64]), cu, max_q, 64)
    got = paged_int4_attention(q, cache, table[:, :4], ints([10 ** 9, 64]), cu, max_q, 10 ** 9)
    assert torch.equal(got, want)
    out = torch.full_like(q, 5.0)
    paged_int4_attention(q, cache, table, ints([-5, 64]), cu, max_q, 100, out=out)
    assert not out[:3].any() and torch.equal(out[3:], want[3:])
    for bad in ([-2 ** 31, 2, 5], [0, 2 ** 31 - 1, 5], [7, 3, 1], [0, -9, 2 ** 31 - 1]):
        out.fill_(5.0)
        paged_int4_attention(q, cache, table, lens, ints(bad), max_q, 100, out=out)
        load_int4(cache, table, ints(bad), 9)
    torch.cuda.synchronize()


def test_the_same_page_in_several_sequences():
    """A shared prefix: table rows that name the same pages."""
    c = Call([100, 100, 64], [1, 1, 2], 4, 2, 64, seed=10)
    c.table[1] = c.table[0]
    c.table[2, :4] = c.table[0, :4]
    c.check()


def test_another_stream_and_graphs():
    """On a side stream; captured twice, each replayed between eager calls on changed inputs."""
    c = Call([3000, 700, 90], [1, 2, 1], 6, 2, 128, page=64, seed=12)
    q, cache, table, lens, cu, max_q, max_k = c.device_args()
    eager = paged_int4_attention(q, cache, table, lens, cu, max_q, max_k)
    c.check(eager)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = paged_int4_attention(q, cache, table, lens, cu, max_q, max_k)
    side.synchronize()
    assert torch.equal(other, eager)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = paged_int4_attention(q, cache, table, lens, cu, max_q, max_k)
        graphs.append((graph, out))
    for step in range(4):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(step)).half())
        lens.copy_(ints([3000 - 500 * step, 700 - step, 90 + 0 * step]))
        want = paged_int4_attention(q, cache, table, lens, cu, max_q, max_k)
        for graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, out in graphs)


def test_a_serving_step_in_a_graph():
    """extend, store and attention together: prompts are admitted, then decode steps replay one graph;
    every step against the definition, then the sequences leave."""
    heads, hk, dim, page, pages, batch = 4, 2, 64, 16, 24, 3
    tables = PageTables.empty(pages, batch, 6, page)
    cache = PagedInt4Cache.empty(pages, hk, dim, page)
    for t in (cache.k_codes, cache.v_codes):
        t.fill_(255)
    for t in (cache.k_params, cache.v_params):
        t.fill_(float("nan"))
    gen = torch.Generator().manual_seed(3)
    history = [[np.zeros((0, hk, dim))] * 2 for _ in range(batch)]

    def step(new, q, k, v, tokens):
        plan = tables.extend(new, tokens)
        store_int4(k, v, cache, plan.slots)
        out = paged_int4_attention(q, cache, tables.block_table, tables.seq_lens, plan.cu_seqlens, tokens, 96)
        return plan, out

    def make(tokens):
        return [torch.randn(tokens, h, dim, generator=gen).half().cuda() for h in (heads, hk, hk)]

    def check(plan, out, new, q, k, v):
        cu = plan.cu_seqlens.tolist()
        for b in range(batch):
            for j, x in ((0, k), (1, v)):
                codes, params = P.quantise(x[cu[b]:cu[b + 1]].double().cpu().numpy())
                history[b][j] = np.concatenate([history[b][j], P.dequantise(codes, params, dim)])
        pool = [a.cpu().numpy() for a in (cache.k_codes, cache.k_params, cache.v_codes, cache.v_params)]
        lens, table = tables.seq_lens.tolist(), tables.block_table.cpu().numpy()
        assert lens == [len(h[0]) for h in history]
        ref, mag, size = P.attention(q.double().cpu().numpy(), *pool, dim, table, lens, cu, max(new), 96, True, dim ** -0.5)
        assert (np.abs(out.double().cpu().numpy() - ref) <= tolerance(ref, mag, size, dim, "fp16")).all()
        got = load_int4(cache, tables.block_table, ints(np.concatenate([[0], np.cumsum(lens)]).tolist()), sum(lens))
        for j in (0, 1):
            assert np.array_equal(got[j].double().cpu().numpy(), np.concatenate([h[j] for h in history]))

    new = [20, 33, 1]
    q, k, v = make(sum(new))
    plan, out = step(ints(new), q, k, v, sum(new))
    check(plan, out, new, q, k, v)
    one, (q, k, v) = ints([1] * batch), make(batch)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, out = step(one, q, k, v, batch)
    for _ in range(20):
        for t, fresh in zip((q, k, v), make(batch)):
            t.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        check(plan, out, [1] * batch, q, k, v)
    tables.truncate(ints([0] * batch))
    assert int(tables.free_count) == pages and sorted(tables.free_pages.tolist()) == list(range(pages))
    assert (tables.block_table == -1).all() and not tables.seq_lens.any()
