"""Refusals of the paged 4-bit KV cache (CPU): the Python calls raise before any launch, on the shapes
and types first and then on the device; the C ABI returns an error; the library's structs match
their mirrors; the oracle's quantisation keeps its bounds."""
from __future__ import annotations

import ctypes
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from _paged_int4 import make_pool
from oracle import paged_int4_oracle as P
from tilemix_amd import _native
from tilemix_amd.attention.hip.paged_int4 import (PagedInt4Cache, PageTables, load_int4, paged_int4_attention,
                                                  store_int4)

HEADER = Path(__file__).resolve().parents[1] / "include" / "tilemix_hip.h"


def cache(pages=3, heads=2, dim=64, page=16):
    return PagedInt4Cache(*(torch.from_numpy(a) for a in make_pool(pages, heads, dim, page)), dim)


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


def half(*shape):
    return torch.zeros(shape, dtype=torch.float16)


# ---- the cache ------------------------------------------------------------------------


def test_cache_shapes():
    c = cache(pages=5, heads=3, dim=80, page=48)
    assert (c.pages, c.heads, c.page_size, c.head_dim) == (5, 3, 48, 80)
    assert c.k_codes.shape == (5, 3, 48, 48) and c.v_params.shape == (5, 3, 48, 3, 2)
    e = PagedInt4Cache.empty(5, 3, 80, 48, device="cpu")
    assert all(a.shape == b.shape and a.dtype == b.dtype for a, b in zip(e._args[:4], c._args[:4]))


def test_cache_refuses():
    c = cache()
    good = list(c._args)

    def refused(error, match, **changed):
        names = ("k_codes", "k_params", "v_codes", "v_params", "head_dim")
        args = [changed.get(n, g) for n, g in zip(names, good)]
        with pytest.raises(error, match=match):
            PagedInt4Cache(*args)

    refused(TypeError, "k_codes must be Byte", k_codes=c.k_codes.to(torch.int8))
    refused(TypeError, "v_params must be Half", v_params=c.v_params.float())
    refused(TypeError, "v_codes must be a torch.Tensor", v_codes=[1])
    refused(ValueError, "head_dim must be in", head_dim=129)
    refused(ValueError, "head_dim must be in", head_dim=0)
    refused(ValueError, "k_codes must be", head_dim=65)
    refused(ValueError, "k_codes must be", k_codes=c.k_codes[0])
    refused(ValueError, "k_codes must be", k_codes=c.k_codes[:0])
    refused(ValueError, "multiple of 16", k_codes=c.k_codes[:, :, :15].contiguous())
    refused(ValueError, "v_codes does not match", v_codes=c.v_codes[:2])
    refused(ValueError, "k_params does not match", k_params=c.k_params[..., :1, :])
    refused(ValueError, "k_codes must be contiguous", k_codes=c.k_codes.transpose(0, 1).contiguous().transpose(0, 1))
    odd = torch.zeros(c.v_codes.numel() + 1, dtype=torch.uint8)[1:].view(c.v_codes.shape)
    refused(ValueError, "v_codes must be contiguous and aligned", v_codes=odd)
    for page in (0, 8, 24):
        with pytest.raises(ValueError, match="page_size"):
            PagedInt4Cache.empty(2, 2, 64, page, device="cpu")
    with pytest.raises(TypeError):
        PagedInt4Cache(*good[:4], 64.0)


# ---- calls ------------------------------------------------------------------------------


def test_store_refuses():
    c, k, slots = cache(), half(4, 2, 64), torch.zeros(4, dtype=torch.int64)
    for error, match, args in (
            (TypeError, "k must be float16 or bfloat16", (k.float(), k.float(), slots)),
            (TypeError, "v must be Half", (k, k.bfloat16(), slots)),
            (ValueError, "k must be", (k[:, :1], k[:, :1], slots)),
            (ValueError, "k must be", (k[..., :32], k[..., :32], slots)),
            (ValueError, "k must be", (k[0], k[0], slots)),
            (ValueError, "one shape", (k, k[:3], slots)),
            (TypeError, "slots must be Long", (k, k, slots.int())),
            (ValueError, "slots must be a vector of 4", (k, k, slots[:3])),
            (ValueError, "slots must be a vector", (k, k, slots[:, None])),
            (TypeError, "k must be a torch.Tensor", (None, k, slots)),
            (TypeError, "plain strided", (k.to_sparse(), k, slots)),
            (RuntimeError, "GPU", (k, k, slots))):
        with pytest.raises(error, match=match):
            store_int4(args[0], args[1], c, args[2])


def test_load_refuses():
    c, table, cu = cache(), torch.zeros(2, 3, dtype=torch.int32), ints(0, 4, 9)
    for error, match, args in (
            (TypeError, "block_table must be Int", (table.long(), cu, 9)),
            (ValueError, "block_table must be", (table[0], cu, 9)),
            (TypeError, "cu_seqlens must be Int", (table, cu.long(), 9)),
            (ValueError, "cu_seqlens must be a vector of 3", (table, cu[:2], 9)),
            (ValueError, "num_tokens must be in", (table, cu, -1)),
            (TypeError, "integer", (table, cu, 9.0)),
            (TypeError, "dtype must be float16 or bfloat16", (table, cu, 9, torch.float32)),
            (TypeError, "dtype must be a torch.dtype", (table, cu, 9, "fp16")),
            (ValueError, "without a sequence", (table[:0], cu[:1], 9)),
            (RuntimeError, "GPU", (table, cu, 9))):
        with pytest.raises(error, match=match):
            load_int4(c, *args)


def test_attention_refuses():
    c, q, table, lens, cu = cache(), half(5, 6, 64), torch.zeros(2, 3, dtype=torch.int32), ints(8, 9), ints(0, 2, 5)
    good = dict(q=q, block_table=table, seq_lens=lens, cu_seqlens_q=cu, max_seqlen_q=3, max_seqlen_k=9)
    for error, match, changed in (
            (TypeError, "q must be float16 or bfloat16", dict(q=q.float())),
            (ValueError, "q must be", dict(q=q[..., :32])),
            (ValueError, "q must be", dict(q=q[None])),
            (ValueError, "multiple of the cache's 2", dict(q=q[:, :5])),
            (ValueError, "multiple of the cache's 2", dict(q=q[:, :0])),
            (TypeError, "block_table must be Int", dict(block_table=table.long())),
            (ValueError, "seq_lens must be a vector of 2", dict(seq_lens=ints(1))),
            (TypeError, "seq_lens must be Int", dict(seq_lens=lens.long())),
            (ValueError, "cu_seqlens_q must be a vector of 3", dict(cu_seqlens_q=cu[:2])),
            (ValueError, "without cu_seqlens_q", dict(cu_seqlens_q=None)),
            (ValueError, "max_seqlen_q must be in", dict(max_seqlen_q=-1)),
            (ValueError, "max_seqlen_k must be in", dict(max_seqlen_k=2 ** 31)),
            (TypeError, "integer", dict(max_seqlen_k=9.5)),
            (TypeError, "real number", dict(sm_scale="x")),
            (TypeError, "out must be Half", dict(out=q.bfloat16())),
            (ValueError, "out must have q's shape", dict(out=q[:4])),
            (ValueError, "out must have q's shape", dict(out=half(1, 6, 64).expand(5, 6, 64))),
            (ValueError, "out must have q's shape", dict(out=half(5, 6, 128)[..., ::2])),
            (RuntimeError, "GPU", {})):
        args = {**good, **changed}
        with pytest.raises(error, match=match):
            paged_int4_attention(args.pop("q"), c, args.pop("block_table"), args.pop("seq_lens"),
                                 args.pop("cu_seqlens_q"), args.pop("max_seqlen_q"), args.pop("max_seqlen_k"), **args)


def test_attention_refuses_rows_that_overlap_and_endless_scales():
    c, table, lens = cache(), torch.zeros(5, 3, dtype=torch.int32), ints(8, 9, 1, 2, 3)
    room = half(9, 6, 64)
    q = room[2:7]
    flat = half(5 * 6 * 64 + 64)
    for match, changed in (
            ("rows that lie apart", dict(out=flat.as_strided((5, 6, 64), (6 * 64, 63, 1)))),
            ("rows that lie apart", dict(out=flat.as_strided((5, 6, 64), (5 * 64, 64, 1)))),
            ("rows that lie apart", dict(out=flat.as_strided((5, 6, 64), (64, 4 * 64, 1)))),
            ("q itself or have memory of its own", dict(out=room[1:6])),
            ("sm_scale must be finite", dict(sm_scale=float("nan"))),
            ("sm_scale must be finite", dict(sm_scale=1e39)),
            ("sm_scale must be finite", dict(sm_scale=-float("inf")))):
        with pytest.raises(ValueError, match=match):
            paged_int4_attention(q, c, table, lens, None, 1, 9, **changed)
    for out in (q, room[:5].clone(), half(6, 5, 64).transpose(0, 1), half(5, 6, 80)[..., 8:72]):
        with pytest.raises(RuntimeError, match="GPU"):
            paged_int4_attention(q, c, table, lens, None, 1, 9, out=out)


def test_tables_refuse():
    t = PageTables.empty(9, 2, 4, 16, device="cpu")
    assert t.free_pages.tolist() == list(range(8, -1, -1)) and t.free_count.tolist() == [9]

    def tables(**changed):
        args = dict(block_table=t.block_table, seq_lens=t.seq_lens, free_pages=t.free_pages, free_count=t.free_count,
                    page_size=16)
        args.update(changed)
        return PageTables(**args)

    for error, match, made, new, tokens in (
            (TypeError, "new lengths must be Int", t, torch.zeros(2, dtype=torch.int64), 4),
            (ValueError, "new lengths must be a vector of 2", t, ints(1), 4),
            (ValueError, "num_tokens must be in", t, ints(1, 2), -1),
            (TypeError, "block_table must be Int", tables(block_table=t.block_table.long()), ints(1, 2), 4),
            (ValueError, "rows of its own", tables(block_table=t.block_table[:1].expand(2, 4)), ints(1, 2), 4),
            (ValueError, "rows of its own", tables(block_table=t.block_table[:, ::2]), ints(1, 2), 4),
            (ValueError, "seq_lens must be a vector of 2", tables(seq_lens=ints(1, 2, 3)), ints(1, 2), 4),
            (ValueError, "contiguous", tables(free_pages=t.free_pages[::2]), ints(1, 2), 4),
            (ValueError, "free_count must be a vector of 1", tables(free_count=ints(1, 2)), ints(1, 2), 4),
            (ValueError, "page_size must be in", tables(page_size=0), ints(1, 2), 4),
            (ValueError, "at most 4096", PageTables.empty(9, 4097, 1, 16, device="cpu"),
             torch.zeros(4097, dtype=torch.int32), 4),
            (ValueError, "without a sequence", PageTables.empty(9, 0, 1, 16, device="cpu"), ints(), 4),
            (RuntimeError, "GPU", t, ints(1, 2), 4)):
        with pytest.raises(error, match=match):
            made.extend(new, tokens)
    with pytest.raises(ValueError, match="vector of 2"):
        t.truncate(ints(1))
    with pytest.raises(RuntimeError, match="GPU"):
        t.truncate(ints(1, 2))


# ---- C ABI --------------------------------------------------------------------------------


@pytest.fixture(scope="module")
def lib():
    return _native.load_library()


def test_struct_sizes_and_fields(lib):
    text = HEADER.read_text()
    for which, struct, cls in ((4, "tilemix_kv4_rows_params", _native.Kv4RowsParams),
                               (5, "tilemix_kv4_attn_params", _native.Kv4AttnParams),
                               (6, "tilemix_kv4_tables_params", _native.Kv4TablesParams)):
        assert lib.tilemix_params_size(which) == ctypes.sizeof(cls)
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), text, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = [n.replace("*", "").strip() for decl in body.split(";") if decl.strip()
                  for n in re.sub(r"^\s*(const\s+)?\w+", "", decl.strip()).split(",")]
        assert [f[0] for f in cls._fields_] == fields
    assert __import__("tilemix_amd._host", fromlist=["x"]).kv4_built_for() == tuple(
        lib.tilemix_params_size(i) for i in (4, 5, 6))


def _pool(p, page_size=16, pages=4, heads=2, head_dim=64):
    for name in ("k_codes", "k_params", "v_codes", "v_params"):
        setattr(p, name, 1 << 20)
    p.pages, p.page_size, p.head_dim = pages, page_size, head_dim
    if hasattr(p, "heads"):
        p.heads = heads
    else:
        p.heads_k = heads
    return p


def test_c_entry_points_refuse(lib):
    """Invalid parameters return before any HIP call (the pointers here are no memory)."""
    err = lambda: lib.tilemix_last_error().decode()
    for name in ("store", "load", "attn", "extend", "truncate"):
        assert getattr(lib, f"tilemix_kv4_{name}")(None, None) == 1 and "null params" in err()
    assert lib.tilemix_kv4_attn_workspace(None) == -1
    rows = _native.Kv4RowsParams
    for fn in (lib.tilemix_kv4_store, lib.tilemix_kv4_load):
        for change in (dict(page_size=8), dict(page_size=0), dict(pages=0), dict(heads=0), dict(heads=65536),
                       dict(head_dim=0), dict(head_dim=129), dict(dtype=2), dict(k_codes=None),
                       dict(v_codes=(1 << 20) + 8), dict(k_params=(1 << 20) + 2), dict(tokens=-1),
                       dict(tokens=1 << 40), dict(tokens=5)):
            p = _pool(rows())
            for k, v in change.items():
                setattr(p, k, v)
            assert fn(ctypes.byref(p), None) == 1, change
        assert fn(ctypes.byref(_pool(rows())), None) == 0  # no row
    p = _pool(rows())
    p.k = p.v = p.cu_seqlens = 1 << 20
    p.tokens = 3
    assert lib.tilemix_kv4_load(ctypes.byref(p), None) == 1 and "no sequence" in err()

    def attn(**change):
        p = _pool(_native.Kv4AttnParams())
        p.heads_q, p.batch, p.table_columns, p.max_seqlen_q, p.max_seqlen_k, p.tokens_q = 6, 2, 1000, 1, 16000, 2
        p.q = p.out = p.block_table = p.seq_lens = 1 << 20
        for k, v in change.items():
            setattr(p, k, v)
        return p

    for change in (dict(heads_q=5), dict(heads_q=0), dict(batch=-1), dict(batch=65536), dict(max_seqlen_q=-1),
                   dict(max_seqlen_k=-1), dict(tokens_q=-1), dict(tokens_q=1 << 31), dict(table_columns=-1),
                   dict(head_dim=200), dict(max_seqlen_q=2 ** 31 - 1),
                   dict(table_columns=2 ** 27, max_seqlen_k=2 ** 30 + 1)):
        assert lib.tilemix_kv4_attn(ctypes.byref(attn(**change)), None) == 1, change
        assert lib.tilemix_kv4_attn_workspace(ctypes.byref(attn(**change))) == -1
    for change in (dict(q=None), dict(out=None), dict(seq_lens=None), dict(block_table=None)):
        assert lib.tilemix_kv4_attn(ctypes.byref(attn(**change)), None) == 1 and "null pointer" in err()
    wanted = lib.tilemix_kv4_attn_workspace(ctypes.byref(attn()))
    assert wanted > 0
    for change in (dict(), dict(workspace=1 << 20, workspace_bytes=wanted - 1),
                   dict(workspace=(1 << 20) + 8, workspace_bytes=wanted)):
        assert lib.tilemix_kv4_attn(ctypes.byref(attn(**change)), None) == 1 and "workspace" in err()
    for change in (dict(batch=0), dict(tokens_q=0), dict(max_seqlen_q=0)):
        assert lib.tilemix_kv4_attn(ctypes.byref(attn(**change)), None) == 0

    def tables(**change):
        p = _native.Kv4TablesParams()
        for name in ("block_table", "seq_lens", "free_pages", "free_count", "ticket", "lens", "slots", "positions",
                     "cu_seqlens", "granted"):
            setattr(p, name, 1 << 20)
        p.batch, p.table_columns, p.page_size, p.free_capacity, p.tokens = 2, 4, 16, 9, 5
        for k, v in change.items():
            setattr(p, k, v)
        return p

    for change in (dict(batch=-1), dict(batch=4097), dict(table_columns=-1), dict(page_size=0), dict(free_capacity=-1),
                   dict(tokens=-1), dict(tokens=1 << 31), dict(seq_lens=None), dict(free_count=None), dict(ticket=None),
                   dict(lens=None), dict(block_table=None), dict(free_pages=None)):
        for fn in (lib.tilemix_kv4_extend, lib.tilemix_kv4_truncate):
            assert fn(ctypes.byref(tables(**change)), None) == 1, change
    for change in (dict(slots=None), dict(positions=None), dict(cu_seqlens=None), dict(granted=None), dict(batch=0)):
        assert lib.tilemix_kv4_extend(ctypes.byref(tables(**change)), None) == 1, change
    assert lib.tilemix_kv4_truncate(ctypes.byref(tables(batch=0)), None) == 0


# ---- the definition ---------------------------------------------------------------------------


def test_quantised_values_are_near():
    """With s' = s + ds and m' = m + dm the rounded parameters: inside the range a code is off by at most half a step
    s'; past its ends (n = 0 or 15, or s' = 0) by |dm| + 15 |ds| more; the value is rounded once.  A rounding to
    fp16 is off by 2^-11 of the value or, below its normal range, by 2^-25."""
    rounding = lambda x: np.maximum(2.0 ** -11 * np.abs(x), 2.0 ** -25)
    rng = np.random.default_rng(0)
    for scale in (1e-6, 1e-2, 1.0, 300.0, 3e4):
        x = (rng.standard_normal((50, 3, 80)) * scale).astype(np.float16).astype(np.float64)
        x[0, 0, 0], x[0, 0, 1] = 65504.0, -65504.0
        codes, params = P.quantise(x)
        y = P.dequantise(codes, params, 80)
        assert np.isfinite(y).all()
        s, m = (np.repeat(params[..., i].astype(np.float64), 32, axis=-1)[..., :80] for i in (0, 1))
        ds = rounding(s) * (1 + 2.0 ** -10)  # of the value before the rounding
        bound = 0.5 * s + rounding(m) * (1 + 2.0 ** -10) + 15 * ds + rounding(y)
        assert (np.abs(y - np.clip(x, -65408, 65408)) <= bound).all()


def test_extreme_groups_stay_finite():
    for a, b in ((-1e9, 1e9), (65504.0, 65504.0), (-65504.0, 65504.0), (-65504.0, -65503.0), (0.0, 6e-8)):
        x = np.linspace(max(a, -65504.0), min(b, 65504.0), 32).astype(np.float16).astype(np.float64)[None]
        x[0, 0], x[0, -1] = a, b
        assert np.isfinite(P.dequantise(*P.quantise(x), 32)).all()
