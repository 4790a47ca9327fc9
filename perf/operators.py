"""Performance cases of the paged 4-bit KV cache: page tables, storing and loading K/V rows,
and the attention that decodes, verifies drafts and continues prompts over the cache.

Format: a (token, KV head) row is split into groups of 32 channels.  A group holds a scale s and a
minimum m in fp16 and a 4-bit code n a channel, and stands for the values fp16(n s + m), where
s = fp16((max - min) / 15), m = fp16(min) and n = clamp(rint((x - m) / s), 0, 15).  Codes are
uint8 [pages, KV heads, page size, width / 2] (the even channel in the low half of a byte),
scales and minima fp16 [pages, KV heads, page size, width / 32, 2]; width is head_dim rounded
up to 32.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"
GROUP = 32
LIMIT = 65408.0  # values are clamped here, so that n s + m stays finite in fp16
OUTLIER_CHANNELS = (7, 33, 70, 101)  # the benchmark's x8 channels of Q and K


# ---- cases ----------------------------------------------------------------------


def _attention(**kw) -> dict:
    """seqs sequences whose caches hold shortest..context tokens, the last new_shortest..new of
    them with a query (one: a decode step)."""
    case = {"kind": "attention", "seqs": 1, "context": 1024, "shortest": 0, "new": 1, "new_shortest": 0,
            "heads": 24, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "float16", "causal": True}
    case.update(kw)
    return case


def _rows(**kw) -> dict:
    """seqs sequences that hold `held` tokens get `new` more stored, and are read back."""
    case = {"kind": "rows", "seqs": 1, "held": 0, "new": 1024, "heads": 8, "dim": 128, "page": 64,
            "dtype": "float16"}
    case.update(kw)
    return case


def _tables(**kw) -> dict:
    """seqs sequences that hold up to `held` tokens are extended by up to `new` and cut back."""
    case = {"kind": "tables", "seqs": 64, "held": 4096, "new": 1, "page": 64}
    case.update(kw)
    return case


def listed() -> list[dict]:
    return [
        # One user of a small model decodes: the latency of a call.
        _attention(name="decode_1x700", context=700, heads=14, kv_heads=2, dim=64, page=16),
        # A serving step: 16 chats of mixed odd lengths.
        _attention(name="decode_16_ragged", seqs=16, context=5000, shortest=61),
        # The largest batch of a decode step.
        _attention(name="decode_64x8192", seqs=64, context=8192),
        # One very long document: the sequence has to be split over the card.
        _attention(name="decode_1x131072", context=131072),
        # bfloat16, seven query heads a KV head, small pages.
        _attention(name="decode_bf16_24_ragged", seqs=24, context=9001, shortest=700, heads=28, kv_heads=4, page=16,
                   dtype="bfloat16"),
        # Drafted tokens are checked: five queries a sequence.
        _attention(name="verify_8x5", seqs=8, context=6144, shortest=1500, new=5, heads=32),
        # A prompt goes on: 512 tokens of it over what the cache holds.
        _attention(name="chunk_512_at_8000", context=8000, new=512),
        # A mixed step: chunks of several prompts and single tokens in one packed call.
        _attention(name="mixed_6", seqs=6, context=4100, shortest=1100, new=1030, new_shortest=1, heads=32, page=32),
        # A short question is appended to a small model's cache and everything is read back.
        _rows(name="rows_37_after_100", held=100, new=37, heads=2, dim=64, page=16),
        # Long prompts enter the cache.
        _rows(name="rows_4x4096", seqs=4, new=4096),
        # Page tables of a decode step.
        _tables(name="tables_step_64"),
        # Page tables when many prompts are admitted at once.
        _tables(name="tables_admit_300", seqs=300, held=0, new=500, page=32),
    ]


def _spread(rng: random.Random, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng: random.Random) -> dict:
    u = rng.random()
    page = rng.choice([16, 32, 64, 128])
    if u < 0.15:
        seqs = _spread(rng, 1, 1024)
        return _tables(seqs=seqs, held=rng.choice([0, _spread(rng, 1, 20000)]),
                       new=rng.choice([1, 1, 5, _spread(rng, 2, max(3, min(8192, 150000 // seqs)))]), page=page)
    dtype = rng.choice(["float16", "float16", "bfloat16"])
    if u < 0.35:
        held = rng.choice([0, 0, _spread(rng, 1, 4000)])
        new = _spread(rng, 1, 16384)
        return _rows(seqs=max(1, min(_spread(rng, 1, 64), 16384 // (held + new))), held=held, new=new,
                     heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 80, 96, 128, 128]), page=page, dtype=dtype)
    heads, kv_heads = rng.choice([(4, 1), (14, 2), (24, 8), (24, 8), (28, 4), (32, 8)])
    context = _spread(rng, 1, 131072)
    seqs = max(1, min(_spread(rng, 1, 64), 400000 // context))
    new = 1 if u < 0.75 else min(context, _spread(rng, 2, 2048))
    while seqs > 1 and seqs * new * context * heads > 512 * 8000 * 24:
        seqs //= 2
    if new * context * heads > 512 * 8000 * 24:
        new = max(2, 512 * 8000 * 24 // (context * heads))
    ragged = seqs > 1 and rng.random() < 0.7
    return _attention(seqs=seqs, context=context, shortest=max(1, context // rng.choice([2, 8, 64])) if ragged else 0,
                      new=new, new_shortest=1 if ragged and new > 1 and rng.random() < 0.5 else 0, heads=heads,
                      kv_heads=kv_heads, dim=rng.choice([64, 80, 96, 128, 128, 128]), page=page, dtype=dtype,
                      causal=rng.random() < 0.9)


def _pick(shortest: int, longest: int, count: int) -> list[int]:
    """`count` lengths shortest..longest, the longest among them (0: all of the longest)."""
    if not shortest:
        return [longest] * count
    rng = random.Random(f"{shortest} {longest} {count}")
    picked = [rng.randint(shortest, longest) for _ in range(count)]
    picked[rng.randrange(count)] = longest
    return picked


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """(tokens in the cache, queries) of each sequence of an attention case."""
    lens = _pick(case["shortest"], case["context"], case["seqs"])
    new = _pick(case["new_shortest"], case["new"], case["seqs"])
    return lens, [min(a, b) for a, b in zip(new, lens)]


def _table_lengths(case: dict) -> tuple[list[int], list[int]]:
    rng = random.Random(f"{case['seqs']} {case['held']} {case['new']}")
    held = [rng.randint(0, case["held"]) if case["held"] else 0 for _ in range(case["seqs"])]
    return held, [rng.randint((case["new"] + 3) // 4, case["new"]) for _ in range(case["seqs"])]


def _width(dim: int) -> int:
    return -(-dim // GROUP) * GROUP


def _row_bytes(dim: int) -> int:
    return _width(dim) // 2 + _width(dim) // GROUP * 4


def work(case: dict) -> dict:
    if case["kind"] == "attention":
        lens, new = _lengths(case)
        pairs = sum(n * length - (n * (n - 1) // 2 if case["causal"] else 0) for length, n in zip(lens, new))
        return {"bytes": 2 * sum(lens) * case["kv_heads"] * _row_bytes(case["dim"])
                + 4 * sum(new) * case["heads"] * case["dim"] + 4 * sum(-(-n // case["page"]) for n in lens),
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    if case["kind"] == "rows":
        stored = case["seqs"] * case["new"] * case["heads"]
        loaded = case["seqs"] * (case["held"] + case["new"]) * case["heads"]
        return {"bytes": 2 * (stored + loaded) * (2 * case["dim"] + _row_bytes(case["dim"])),
                "flops": 2 * (5 * stored + 2 * loaded) * case["dim"]}
    held, new = _table_lengths(case)
    pages = sum(-(-(h + n) // case["page"]) - -(-h // case["page"]) for h, n in zip(held, new))
    # slots and positions in 64 bits; pages taken (read, entered) and given back; lengths
    return {"bytes": 16 * sum(new) + 16 * pages + 4 * 8 * case["seqs"], "flops": 4 * sum(new) + 16 * case["seqs"]}


# ---- inputs -----------------------------------------------------------------------


def _dtype(case: dict) -> torch.dtype:
    return getattr(torch, case["dtype"])


def _int32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _ends(lengths: list[int]) -> torch.Tensor:
    return _int32([0, *np.cumsum(lengths).tolist()])


def _values(gen, shape, outliers: bool) -> torch.Tensor:
    x = torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32)
    if outliers:
        for c in OUTLIER_CHANNELS:
            x[..., c % shape[-1]] *= 8.0
    return x


def _quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and parameters of the rows of x [..., dim] in 32 bits."""
    dim, width = x.shape[-1], _width(x.shape[-1])
    x = x.float().clamp(-LIMIT, LIMIT)
    if width != dim:  # the channels that are not there count as copies of the last one
        x = torch.cat((x, x[..., -1:].expand(*x.shape[:-1], width - dim)), dim=-1)
    x = x.unflatten(-1, (width // GROUP, GROUP))
    low, high = x.amin(-1), x.amax(-1)
    s, m = ((high - low) / 15.0).half(), low.half()
    step = s.float()[..., None]
    n = torch.where(step > 0, (x - m.float()[..., None]) / step, torch.zeros_like(x)).round_().clamp_(0, 15)
    n = n.to(torch.uint8).flatten(-2)
    n[..., dim:] = 0
    return n[..., 0::2] | (n[..., 1::2] << 4), torch.stack((s, m), dim=-1)


def _pool(gen, case: dict, kv_heads: int, pages: int) -> dict:
    """A pool of `pages` pages filled as earlier steps leave it."""
    shape, width = (pages, kv_heads, case["page"]), _width(case["dim"])
    pool = {}
    step = max(1, (1 << 26) // (kv_heads * case["page"] * width))
    for name in ("k", "v"):
        codes = torch.empty((*shape, width // 2), dtype=torch.uint8, device=DEVICE)
        params = torch.empty((*shape, width // GROUP, 2), dtype=torch.float16, device=DEVICE)
        for at in range(0, pages, step):
            n = min(step, pages - at)
            codes[at:at + n], params[at:at + n] = _quantise(
                _values(gen, (n, *shape[1:], case["dim"]), name == "k").to(_dtype(case)))
        pool[f"{name}_codes"], pool[f"{name}_params"] = codes, params
    return pool


def _paged(case: dict, seed: int, lens: list[int]) -> tuple[list[list[int]], int]:
    """Pages of each sequence, in no order, and the number of pages in the pool."""
    needs = [-(-n // case["page"]) for n in lens]
    total = sum(needs) + max(2, sum(needs) // 16)
    order = random.Random(seed).sample(range(total), total)
    rows, at = [], 0
    for n in needs:
        rows.append(order[at:at + n])
        at += n
    return rows, total


def _block_table(rows: list[list[int]], columns: int) -> torch.Tensor:
    table = np.full((len(rows), columns), -1, dtype=np.int32)
    for r, pages in enumerate(rows):
        table[r, :len(pages)] = pages
    return torch.from_numpy(table).to(DEVICE)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = {"case": case}
    if case["kind"] == "tables":
        held, new = _table_lengths(case)
        rows, used = _paged(case, seed, held)
        columns = max(-(-(h + n) // case["page"]) for h, n in zip(held, new)) + 2
        spare = sum(-(-n // case["page"]) + 1 for n in new) + 7
        free = random.Random(seed + 1).sample(range(used, used + spare), spare)
        state.update(block_table=_block_table(rows, columns), seq_lens=_int32(held), held=_int32(held),
                     new_lens=_int32(new), num_tokens=sum(new), free_count=_int32([spare]),
                     free_pages=_int32(free + [page for row in rows for page in row]))
        if own:
            from tilemix_amd.attention.hip.paged_int4 import PageTables
            state["tables"] = PageTables(state["block_table"], state["seq_lens"], state["free_pages"],
                                         state["free_count"], case["page"])
        return state
    if case["kind"] == "rows":
        lens, kv_heads = [case["held"] + case["new"]] * case["seqs"], case["heads"]
    else:
        lens, new = _lengths(case)
        kv_heads = case["kv_heads"]
    rows, pages = _paged(case, seed, lens)
    state.update(_pool(gen, case, kv_heads, pages))
    state["block_table"] = _block_table(rows, max(len(r) for r in rows))
    if case["kind"] == "rows":
        tokens = case["seqs"] * case["new"]
        shape = (tokens, kv_heads, case["dim"])
        state.update(k=_values(gen, shape, True).to(_dtype(case)), v=_values(gen, shape, False).to(_dtype(case)),
                     slots=torch.tensor([row[p // case["page"]] * case["page"] + p % case["page"] for row in rows
                                         for p in range(case["held"], case["held"] + case["new"])], device=DEVICE),
                     cu_seqlens=_ends(lens), num_tokens=sum(lens))
    else:
        state.update(q=_values(gen, (sum(new), case["heads"], case["dim"]), True).to(_dtype(case)),
                     seq_lens=_int32(lens), cu_seqlens_q=_ends(new), max_seqlen_q=max(new), max_seqlen_k=max(lens))
    if own:
        from tilemix_amd.attention.hip.paged_int4 import PagedInt4Cache
        state["cache"] = PagedInt4Cache(state["k_codes"], state["k_params"], state["v_codes"], state["v_params"],
                                        case["dim"])
    return state


# ---- the operators ------------------------------------------------------------------


def run(state: dict):
    return {"attention": _run_attention, "rows": _run_rows, "tables": _run_tables}[state["case"]["kind"]](state)


def _dequantise(codes: torch.Tensor, params: torch.Tensor, dim: int) -> torch.Tensor:
    """The fp16 values of codes [..., width / 2], as fp32 [..., dim]."""
    n = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).unflatten(-1, (-1, GROUP)).float()
    x = n * params[..., 0, None].float() + params[..., 1, None].float()
    return x.half().float().flatten(-2)[..., :dim]


def _run_attention(state: dict) -> torch.Tensor:
    case = state["case"]
    if own:
        from tilemix_amd.attention.hip.paged_int4 import paged_int4_attention
        return paged_int4_attention(state["q"], state["cache"], state["block_table"], state["seq_lens"],
                                    state["cu_seqlens_q"], state["max_seqlen_q"], state["max_seqlen_k"],
                                    causal=case["causal"])
    q, lens, cu = state["q"], state["seq_lens"].long(), state["cu_seqlens_q"].long()
    batch, heads, hk, dim = lens.numel(), case["heads"], case["kv_heads"], case["dim"]
    nq, group, page = state["max_seqlen_q"], heads // hk, case["page"]
    # queries as [batch, KV heads, group * nq, dim], the missing ones zero
    new = cu[1:] - cu[:-1]
    i = torch.arange(nq, device=DEVICE)
    there = i[None, :] < new[:, None]
    at = (cu[:-1, None] + i[None, :]).clamp(max=q.shape[0] - 1)
    x = q[at].float() * there[:, :, None, None]
    x = x.view(batch, nq, hk, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, hk, group * nq, dim)
    table = state["block_table"].long()
    tokens = table.shape[1] * page

    def read(name):
        pages = table.clamp(min=0)
        values = _dequantise(state[f"{name}_codes"][pages], state[f"{name}_params"][pages], dim)
        return values.transpose(1, 2).reshape(batch, hk, tokens, dim)

    scores = torch.matmul(x, read("k").transpose(2, 3).contiguous()) * dim ** -0.5
    j = torch.arange(tokens, device=DEVICE)
    seen = (j[None, None, :] < lens[:, None, None]).expand(batch, nq, tokens)
    if case["causal"]:
        seen = seen & (j[None, None, :] <= (lens - new)[:, None, None] + i[None, :, None])
    scores = scores.view(batch, hk, group, nq, tokens).masked_fill_(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(batch, hk, group * nq, tokens), read("v")).view(batch, hk, group, nq, dim)
    out = out / torch.where(total == 0, torch.ones_like(total), total)
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, nq, heads, dim)
    return out[there].to(q.dtype)


def _run_rows(state: dict):
    case = state["case"]
    if own:
        from tilemix_amd.attention.hip.paged_int4 import load_int4, store_int4
        store_int4(state["k"], state["v"], state["cache"], state["slots"])
        return load_int4(state["cache"], state["block_table"], state["cu_seqlens"], state["num_tokens"],
                         dtype=_dtype(case))
    page, slots, ends = case["page"], state["slots"], state["cu_seqlens"].long()
    t = torch.arange(state["num_tokens"], device=DEVICE)
    seq = torch.searchsorted(ends, t, right=True) - 1
    at = t - ends[seq]
    pages = state["block_table"].long()[seq, at // page]
    out = []
    for name in ("k", "v"):
        codes, params = state[f"{name}_codes"], state[f"{name}_params"]
        codes[slots // page, :, slots % page], params[slots // page, :, slots % page] = _quantise(state[name])
        out.append(_dequantise(codes[pages, :, at % page], params[pages, :, at % page], case["dim"]).to(_dtype(case)))
    return tuple(out)


def _run_tables(state: dict):
    if own:
        tables = state["tables"]
        plan = tables.extend(state["new_lens"], state["num_tokens"])
        tables.truncate(state["held"])
        return (plan.slots, plan.positions, plan.cu_seqlens, plan.granted, tables.block_table, tables.seq_lens,
                tables.free_pages, tables.free_count)
    page, tokens = state["case"]["page"], state["num_tokens"]
    table, lens, new = state["block_table"], state["seq_lens"].long(), state["new_lens"].long()
    free, count = state["free_pages"], state["free_count"].long()
    zero = torch.zeros(1, dtype=torch.int64, device=DEVICE)
    cu = torch.cat((zero, new.cumsum(0)))
    old = (lens + page - 1) // page
    grown = (lens + new + page - 1) // page
    fits = (grown <= table.shape[1]) & (cu[1:] <= tokens)
    needs = torch.where(fits, grown - old, torch.zeros_like(old))
    granted = fits & (needs.cumsum(0) <= count)
    needs = torch.where(granted, needs, torch.zeros_like(needs))
    base = needs.cumsum(0) - needs
    # extend
    column = torch.arange(table.shape[1], device=DEVICE)[None, :]
    taken = (column >= old[:, None]) & (column < (old + needs)[:, None])
    take = (count - 1 - base[:, None] - (column - old[:, None])).clamp(0, free.numel() - 1)
    table = torch.where(taken, free[take], table)
    count = count - needs.sum()
    lens = torch.where(granted, lens + new, lens)
    t = torch.arange(tokens, device=DEVICE)
    seq = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=lens.numel() - 1)
    there = granted[seq] & (t < cu[-1])
    at = state["seq_lens"].long()[seq] + t - cu[seq]
    slot = table[seq, (at // page).clamp(max=table.shape[1] - 1)].long() * page + at % page
    slots = torch.where(there, slot, torch.full_like(slot, -1))
    positions = torch.where(there, at, torch.zeros_like(at))
    # truncate
    kept = torch.minimum(lens, state["held"].long())
    keep = (kept + page - 1) // page
    back = (lens + page - 1) // page - keep
    total, base = back.sum(), back.cumsum(0) - back
    given = (column >= keep[:, None]) & (column < (keep + back)[:, None])
    to = count + total - 1 - base[:, None] - (column - keep[:, None])
    free = torch.cat((free, free[:1]))
    free = free.scatter(0, torch.where(given, to, torch.full_like(to, free.numel() - 1)).flatten(), table.flatten())
    table = torch.where(given, torch.full_like(table, -1), table)
    return (slots, positions, cu.int(), granted.int(), table, kept.int(), free[:-1], (count + total).int())


# ---- 64-bit evaluation ----------------------------------------------------------------


def _exact_values(codes: torch.Tensor, params: torch.Tensor, dim: int) -> torch.Tensor:
    low, high = torch.bitwise_and(codes, 15).double(), torch.bitwise_right_shift(codes, 4).double()
    out = torch.empty((*codes.shape[:-1], codes.shape[-1] * 2), dtype=torch.float64, device=codes.device)
    out[..., 0::2], out[..., 1::2] = low, high
    scale = params[..., 0].double().repeat_interleave(GROUP, dim=-1)
    least = params[..., 1].double().repeat_interleave(GROUP, dim=-1)
    return out.mul_(scale).add_(least).half().double()[..., :dim]


def exact(case: dict, seed: int):
    global own
    kept, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = kept
    return {"attention": _exact_attention, "rows": _exact_rows, "tables": _exact_tables}[case["kind"]](state)


def _exact_attention(state: dict) -> torch.Tensor:
    case = state["case"]
    dim, hk, group = case["dim"], case["kv_heads"], case["heads"] // case["kv_heads"]
    lens, new = _lengths(case)
    out, row = [], 0
    for b, (length, nq) in enumerate(zip(lens, new)):
        pages = state["block_table"][b, :-(-length // case["page"])].long()
        limit = torch.arange(length - nq, length, device=DEVICE) if case["causal"] else torch.full(
            (nq,), length - 1, device=DEVICE)
        hidden = torch.arange(length, device=DEVICE)[None, :] > limit[:, None]
        q = state["q"][row:row + nq].double()
        result = torch.empty_like(q)
        for h in range(hk):
            k, v = (_exact_values(state[f"{n}_codes"][pages, h], state[f"{n}_params"][pages, h], dim).reshape(
                -1, dim)[:length] for n in ("k", "v"))
            for g in range(h * group, (h + 1) * group):
                scores = (q[:, g] @ k.T) / math.sqrt(dim)
                scores.masked_fill_(hidden, float("-inf"))
                result[:, g] = torch.softmax(scores, dim=-1) @ v
        out.append(result)
        row += nq
    return torch.cat(out)


def _exact_rows(state: dict):
    case = state["case"]
    page, dim, width = case["page"], case["dim"], _width(case["dim"])
    held, new = case["held"], case["new"]
    out = []
    for name in ("k", "v"):
        result = torch.empty((case["seqs"], held + new, case["heads"], dim), dtype=torch.float64, device=DEVICE)
        fresh = state[name].double().view(case["seqs"], new, case["heads"], dim).clamp(-LIMIT, LIMIT)
        for c in range(0, width, GROUP):
            x = fresh[..., c:min(dim, c + GROUP)]
            least, most = x.min(dim=-1, keepdim=True).values, x.max(dim=-1, keepdim=True).values
            s, m = ((most - least) / 15).half().double(), least.half().double()
            n = torch.clamp(torch.round((x - m) / torch.where(s == 0, torch.ones_like(s), s)), 0, 15)
            n = torch.where(s == 0, torch.zeros_like(n), n)
            result[:, held:, :, c:c + x.shape[-1]] = (n * s + m).half().double()
        for b in range(case["seqs"] if held else 0):
            pages = state["block_table"][b, :-(-held // page)].long()
            old = _exact_values(state[f"{name}_codes"][pages], state[f"{name}_params"][pages], dim)
            result[b, :held] = old.transpose(1, 2).reshape(-1, case["heads"], dim)[:held]
        out.append(result.flatten(0, 1))
    return tuple(out)


def _exact_tables(state: dict):
    """The definition step by step: every request takes its pages from the top of the stack, one
    after the other, and the last page taken goes back first."""
    page, tokens = state["case"]["page"], state["num_tokens"]
    table = state["block_table"].tolist()
    lens, new, held = (state[n].tolist() for n in ("seq_lens", "new_lens", "held"))
    stack = state["free_pages"].tolist()
    count = state["free_count"].item()
    slots, positions, cu, granted, short = [-1] * tokens, [0] * tokens, [0], [], False
    for b, n in enumerate(new):
        old, grown, start = -(-lens[b] // page), -(-(lens[b] + n) // page), cu[-1]
        cu.append(start + n)
        fits = grown <= len(table[b]) and cu[-1] <= tokens
        short = short or (fits and grown - old > count)
        ok = fits and (not short or grown == old)
        granted.append(int(ok))
        if not ok:
            continue
        for c in range(old, grown):
            count -= 1
            table[b][c] = stack[count]
        for i in range(n):
            at = lens[b] + i
            slots[start + i], positions[start + i] = table[b][at // page] * page + at % page, at
        lens[b] += n
    for b in reversed(range(len(lens))):
        kept = min(lens[b], held[b])
        for c in reversed(range(-(-kept // page), -(-lens[b] // page))):
            stack[count] = table[b][c]
            table[b][c] = -1
            count += 1
        lens[b] = kept
    long = [torch.tensor(x, device=DEVICE) for x in (slots, positions)]
    return (*long, _int32(cu), _int32(granted), _int32(table), _int32(lens), _int32(stack), _int32([count]))
